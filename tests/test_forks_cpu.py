"""Forks of running requests under a short pool, and what forks and compaction may touch, on the CPU."""
import dataclasses

import numpy as np
import pytest
import torch

from vllm_suffix_hybrid_b200.engine.config import CacheConfig, EngineConfig, SpecConfig, llama3_8b_config, shrink
from vllm_suffix_hybrid_b200.engine.llm import LLMEngine


def engine(blocks=0, method="none", kv="nvfp4", seqs=4, budget=4096, asynchronous=False, chunked=True):
    m = dataclasses.replace(shrink(llama3_8b_config(), layers=2, hidden=128, vocab=256), kv_format=kv, dtype="float32")
    return LLMEngine(EngineConfig(model=m, spec=SpecConfig(method=method, k=3, async_scheduling=asynchronous),
                                  cache=CacheConfig(max_model_len=1024, num_blocks=blocks), max_num_seqs=seqs, device="cpu",
                                  cuda_graphs=False, max_prefill_tokens=budget, chunked_prefill=chunked))


def drain(eng, steps=3000):
    for _ in range(steps):
        if not eng.has_work():
            return
        eng.step()
    raise AssertionError("requests are left")


# ----------------------------------------------------------------------------------------------- a short pool
@pytest.mark.parametrize("kv", ["nvfp4", "bf16"])
@pytest.mark.parametrize("budget", [4096, 64])
def test_a_fork_behind_a_request_that_does_not_fit_runs_first(kv, budget):
    """The waiting fork holds its parent's blocks: once nothing runs they are all that the larger request lacks."""
    rng = np.random.default_rng(1)
    prompt, large = rng.integers(0, 256, 400), rng.integers(0, 256, 600)
    eng = engine(14, kv=kv, budget=budget)
    free = eng.pool.free
    a = eng.add_request(prompt, max_new_tokens=20)
    while not eng.running:
        eng.step()
    b = eng.add_request(large, max_new_tokens=20)
    eng.step()
    sofar = list(eng.running[0].output)
    c = eng.fork_request(a, [5, 6], max_new_tokens=30)
    drain(eng)
    assert eng.pool.free == free
    want = engine(kv=kv, budget=budget)
    assert eng.finished[b].output == want.generate([large], 20)[0]
    assert eng.finished[c].output == want.generate([np.concatenate([prompt, sofar, [5, 6]])], 30)[0]


@pytest.mark.parametrize("chunked", [True, False])
def test_forks_that_do_not_fit_beside_each_other_give_their_blocks_up(chunked):
    """Two forks that each need more than is free while the other waits: the later one prefills its prompt anew."""
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 256, n) for n in (300, 290)]
    eng = engine(14, chunked=chunked)
    free = eng.pool.free
    ids = [eng.add_request(p, max_new_tokens=8) for p in prompts]
    while len(eng.running) < 2:
        eng.step()
    sofar = [list(r.output) for r in eng.running]
    kids = [eng.fork_request(i, [7, 8], max_new_tokens=340) for i in ids]  # 11 blocks each, 5 of them held
    drain(eng)
    assert eng.pool.free == free
    want = engine()
    for i, (kid, p, s) in enumerate(zip(kids, prompts, sofar)):
        assert eng.finished[kid].output == want.generate([np.concatenate([p, s, [7, 8]])], 340)[0], i


def test_a_fork_too_large_for_the_pool_is_refused_when_its_turn_comes():
    eng = engine(8)
    a = eng.add_request(np.arange(300) % 256, max_new_tokens=6)
    eng.step()
    b = eng.fork_request(a, max_new_tokens=400)
    with pytest.raises(MemoryError, match=b):
        drain(eng)
    assert a in eng.finished
    assert eng.abort_request(b)
    assert eng.pool.free == 7 and not eng.has_work()


@pytest.mark.parametrize("asynchronous", [True, False])
def test_a_fork_takes_no_block_that_is_promised(asynchronous):
    """Two requests that fill the pool in the end: at no step is there a block for a fork's copy."""
    eng = engine(10, method="suffix", seqs=3, asynchronous=asynchronous)
    a = eng.add_request(np.arange(50) % 256, max_new_tokens=126)  # with the look-ahead three blocks to the token
    b = eng.add_request(np.arange(60) % 256, max_new_tokens=300)  # six
    eng.step()
    parent = next(r for r in eng.running if r.rid == b)
    while a not in eng.finished:
        assert eng._unclaimed_blocks() == 0
        if parent.committed % 64:  # (a whole block is shared, not copied)
            with pytest.raises(MemoryError, match="unpromised"):
                eng.fork_request(b, max_new_tokens=2)
        for _ in range(3):
            eng.step()
        eng._drain()
    drain(eng)
    assert len(eng.finished[b].output) == 300 and eng.pool.free == 9


@pytest.mark.parametrize("method", ["suffix", "hybrid"])
def test_pipelined_steps_stay_within_their_reservations(method):
    """Every length at which the pipeline's look-ahead crosses into a new block, in a pool that the requests fill."""
    eng = engine(10, method=method, seqs=3, asynchronous=True)
    assert eng._async
    rng = np.random.default_rng(4)
    for n in range(100, 164, 3):
        ids = [eng.add_request(rng.integers(0, 256, n), max_new_tokens=20) for _ in range(3)]
        while eng.has_work():
            eng.step()
            assert eng._unclaimed_blocks() >= 0
            assert all(len(r.blocks) <= eng._reservation(r) for r in eng.running)
        assert all(len(eng.finished[i].output) == 20 for i in ids)


# ----------------------------------------------------------------------------------------------- what is copied
def test_forks_and_compaction_refuse_a_cache_that_is_not_laid_out_by_blocks():
    """A cache tensor that page copies do not know would keep another request's rows without a word."""
    eng = engine()
    a = eng.add_request(np.arange(100) % 256, max_new_tokens=8)
    b = eng.add_request(np.arange(90) % 256, max_new_tokens=8)
    eng.step()
    free = eng.pool.free
    eng.caches.append((torch.zeros(eng.pool.num_blocks + 1, 64),))
    with pytest.raises(ValueError, match="laid out by blocks"):
        eng.fork_request(a, max_new_tokens=2)
    assert eng.pool.free == free and not eng.waiting
    eng.caches.pop()
    eng.fork_request(a, max_new_tokens=2)
    eng.abort_request(a)
    eng.caches.append((torch.zeros(eng.pool.num_blocks + 1, 64),))
    with pytest.raises(ValueError, match="laid out by blocks"):
        eng.compact_cache()
    eng.caches.pop()
    eng.compact_cache()
    drain(eng)
    assert len(eng.finished[b].output) == 8
