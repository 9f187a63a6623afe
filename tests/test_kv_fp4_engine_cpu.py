"""The 4-bit KV cache in the engine, forks of a running request and cache compaction, on the CPU."""
import dataclasses

import numpy as np
import pytest
import torch

from vllm_suffix_hybrid_b200.engine.config import (CacheConfig, EngineConfig, SpecConfig, deepseek_v32_config,
                                                   llama3_8b_config, qwen3_next_config, shrink)
from vllm_suffix_hybrid_b200.engine.kv_cache import BlockPool
from vllm_suffix_hybrid_b200.engine.llm import LLMEngine

BASE = {"llama": llama3_8b_config, "qwen3_next": qwen3_next_config, "deepseek_v32": deepseek_v32_config}


def engine(name="llama", kv="nvfp4", method="none", seqs=4, budget=4096, **model):
    m = shrink(BASE[name](), layers=2, hidden=128, vocab=256)
    m = dataclasses.replace(m, kv_format=kv, **model)
    return LLMEngine(EngineConfig(model=m, spec=SpecConfig(method=method, k=3), cache=CacheConfig(max_model_len=512),
                                  max_num_seqs=seqs, device="cpu", cuda_graphs=False, max_prefill_tokens=budget))


def drain(eng):
    while eng.has_work():
        eng.step()


@pytest.mark.parametrize("name", ["llama", "qwen3_next"])
@pytest.mark.parametrize("method", ["none", "hybrid", "suffix"])
def test_generates_on_a_4bit_cache_a_quarter_the_size(name, method):
    eng = engine(name, method=method)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 256, n) for n in (5, 70, 64)]
    outs = eng.generate(prompts, max_new_tokens=8)
    assert all(len(o) == 8 for o in outs)
    full = engine(name, kv="bf16")
    d, hk = eng.cfg.model.head_dim, eng.model.kv_heads_local
    assert eng.model.kv_block_bytes(64) == 2 * hk * 64 * (d // 2 + d // 16)
    assert full.model.kv_block_bytes(64) == 2 * hk * 64 * d * full.model.embed.element_size()


def test_chunked_prefill_reads_the_cached_prefix():
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, 256, 170)
    assert engine(budget=48).generate([prompt], 10) == engine().generate([prompt], 10)


def test_speculation_changes_no_token(monkeypatch):
    """Batch-invariant greedy decoding: a verify window gives what single tokens give, on the 4-bit cache too."""
    monkeypatch.setenv("SH_BATCH_INVARIANT", "1")
    rng = np.random.default_rng(3)
    prompts = [np.tile(rng.integers(0, 256, 7), 9) for _ in range(3)]
    assert engine(method="suffix").generate(prompts, 24) == engine(method="none").generate(prompts, 24)


def test_the_environment_selects_the_cache_format(monkeypatch):
    monkeypatch.setenv("SUFFIX_HYBRID_KV_FORMAT", "nvfp4")
    assert engine(kv="bf16").caches[0][0].dtype == torch.uint8
    monkeypatch.setenv("SUFFIX_HYBRID_KV_FORMAT", "other")
    assert engine(kv="bf16").caches[0][0].dtype != torch.uint8


def test_unsupported_shapes_are_refused():
    with pytest.raises(ValueError, match="head_dim"):
        engine(head_dim=96)


# ----------------------------------------------------------------------------------------------- forks
@pytest.mark.parametrize("name,kv", [("llama", "nvfp4"), ("llama", "bf16"), ("deepseek_v32", "bf16")])
@pytest.mark.parametrize("length", [20, 63, 64, 130])
def test_a_fork_generates_what_a_fresh_request_generates(name, kv, length):
    rng = np.random.default_rng(length)
    prompt, extra = rng.integers(0, 256, length), [7, 8, 9]
    eng = engine(name, kv)
    free = eng.pool.free
    parent = eng.add_request(prompt, max_new_tokens=12)
    for _ in range(4):
        eng.step()
    sofar = list(eng.running[0].output)
    held = free - eng.pool.free
    child = eng.fork_request(parent, extra, max_new_tokens=6)
    twin = eng.fork_request(parent, max_new_tokens=6)
    committed = length + len(sofar) - 1
    # two copies of a partly filled block, nothing else
    assert free - eng.pool.free == held + (2 if committed % 64 else 0)
    drain(eng)
    assert eng.pool.free == free
    want = engine(name, kv)
    assert eng.finished[child].output == want.generate([np.concatenate([prompt, sofar, extra])], 6)[0]
    assert eng.finished[parent].output == want.generate([prompt], 12)[0]
    assert eng.finished[twin].output == eng.finished[parent].output[len(sofar):len(sofar) + 6]


def test_a_fork_outlives_its_parent_and_can_be_forked_and_aborted():
    eng = engine(method="hybrid")
    free = eng.pool.free
    a = eng.add_request(np.arange(150) % 256, max_new_tokens=30)
    eng.step()
    b = eng.fork_request(a, [1, 2], max_new_tokens=20)
    c = eng.fork_request(a, [3], max_new_tokens=20)
    assert eng.abort_request(c) and eng.abort_request(a)  # c still waits, a runs
    assert eng.pool.free < free
    while not any(r.rid == b for r in eng.running):
        eng.step()
    d = eng.fork_request(b, [5], max_new_tokens=4)
    drain(eng)
    assert len(eng.finished[b].output) == 20 and len(eng.finished[d].output) == 4
    assert eng.pool.free == free


def test_a_fork_waits_for_blocks_like_any_request():
    eng = engine(seqs=2)
    a = eng.add_request(np.arange(100) % 256, max_new_tokens=40)
    b = eng.add_request(np.arange(90) % 256, max_new_tokens=10)
    eng.step()
    c = eng.fork_request(a, max_new_tokens=5)  # both rows are taken
    eng.step()
    assert any(r.rid == c for r in eng.waiting)
    drain(eng)
    assert len(eng.finished[c].output) == 5 and len(eng.finished[b].output) == 10


def test_fork_refusals():
    eng = engine()
    with pytest.raises(ValueError, match="not running"):
        eng.fork_request("nobody")
    a = eng.add_request(np.arange(10), max_new_tokens=5)
    with pytest.raises(ValueError, match="not running"):
        eng.fork_request(a)  # still waiting
    eng.step()
    with pytest.raises(ValueError):
        eng.fork_request(a, max_new_tokens=10_000)
    with pytest.raises(ValueError, match="duplicate"):
        eng.fork_request(a, new_rid=a)
    free = eng.pool.free
    drain(eng)
    assert eng.pool.free > free  # the refused forks held nothing
    q = engine("qwen3_next")
    r = q.add_request(np.arange(10), max_new_tokens=5)
    q.step()
    with pytest.raises(ValueError, match="attention-only"):
        q.fork_request(r)


# ----------------------------------------------------------------------------------------------- compaction
@pytest.mark.parametrize("kv", ["nvfp4", "bf16"])
def test_compaction_moves_live_blocks_down_and_changes_no_token(kv):
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, 256, n) for n in (130, 200, 70, 140)]

    def run(compact):
        eng = engine("llama", kv, method="hybrid")
        free = eng.pool.free
        ids = [eng.add_request(p, max_new_tokens=20) for p in prompts]
        eng.step()
        eng.step()
        child = eng.fork_request(ids[3], [4, 5], max_new_tokens=8)
        eng.abort_request(ids[0])
        eng.abort_request(ids[2])
        if compact:
            n = eng.compact_cache()
            used = {b for r in eng.running + eng.waiting for b in r.blocks}
            assert used == set(range(1, n + 1))
            assert eng.compact_cache() == n and eng.pool.compaction() == {}
        drain(eng)
        assert eng.pool.free == free
        return [eng.finished[i].output for i in ids + [child]]

    assert run(True) == run(False)


def test_pool_counts_holders():
    pool = BlockPool(6)
    a = pool.allocate(3)
    pool.share(a[:2])
    pool.release(a)
    assert pool.free == 3
    assert pool.compaction() == {}
    pool.release(a[:2])
    assert pool.free == 5
    with pytest.raises(ValueError):
        pool.release(a[:1])
    with pytest.raises(ValueError):
        pool.share([5])
    with pytest.raises(MemoryError):
        pool.allocate(6)
