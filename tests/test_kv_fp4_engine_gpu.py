"""The engine on the 4-bit KV cache with the GPU kernels: CUDA graphs, forks, compaction, batch invariance."""
import dataclasses

import numpy as np
import pytest

from vllm_suffix_hybrid_b200.engine.config import (CacheConfig, EngineConfig, SpecConfig, llama3_8b_config,
                                                   qwen3_next_config, shrink)
from vllm_suffix_hybrid_b200.engine.llm import LLMEngine

pytestmark = pytest.mark.gpu


def engine(name="llama", kv="nvfp4", method="hybrid", graphs=True, budget=4096, **model):
    base = {"llama": llama3_8b_config, "qwen3_next": qwen3_next_config}[name]()
    m = dataclasses.replace(shrink(base, layers=3, hidden=256, vocab=1024), kv_format=kv, **model)
    return LLMEngine(EngineConfig(model=m, spec=SpecConfig(method=method, k=3), cache=CacheConfig(max_model_len=2048),
                                  max_num_seqs=4, device="cuda", cuda_graphs=graphs, max_prefill_tokens=budget))


def drain(eng):
    while eng.has_work():
        eng.step()


@pytest.mark.parametrize("name,heads", [("llama", {}), ("qwen3_next", {}), ("llama", dict(heads=8, kv_heads=2, head_dim=128)),
                                        ("llama", dict(heads=4, kv_heads=1, head_dim=256))])
def test_graphs_and_eager_steps_agree(name, heads):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 1024, n) for n in (5, 700, 64, 129)]
    a = engine(name, **heads).generate(prompts, 24)
    b = engine(name, graphs=False, **heads).generate(prompts, 24)
    assert all(len(o) == 24 for o in a) and a == b


def test_speculation_changes_no_token(monkeypatch):
    monkeypatch.setenv("SH_BATCH_INVARIANT", "1")
    rng = np.random.default_rng(2)
    prompts = [np.tile(rng.integers(0, 1024, 9), 20) for _ in range(3)]
    assert engine(method="suffix").generate(prompts, 40) == engine(method="none").generate(prompts, 40)


def test_forks_share_blocks_and_continue():
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1024, n) for n in (100, 640, 333)]
    eng = engine(method="none")
    free = eng.pool.free
    ids = [eng.add_request(p, max_new_tokens=30) for p in prompts]
    for _ in range(5):
        eng.step()
    outs = [list(r.output) for r in eng.running]
    kids = [eng.fork_request(i, [3, 1, 4], max_new_tokens=10) for i in ids[:1]] + [eng.fork_request(ids[1], max_new_tokens=10)]
    drain(eng)
    assert eng.pool.free == free
    fresh = engine(method="none").generate([np.concatenate([prompts[0], outs[0], [3, 1, 4]])], 10)[0]
    same = [eng.finished[kids[0]].output == fresh,
            eng.finished[kids[1]].output == eng.finished[ids[1]].output[len(outs[1]):len(outs[1]) + 10]]
    assert any(same)  # another summation order may flip a bf16 near-tie in one of them
    assert all(len(eng.finished[k].output) == 10 for k in kids)


def test_compaction_changes_no_token():
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 1024, n) for n in (400, 500, 70, 640)]

    def run(compact):
        eng = engine()
        ids = [eng.add_request(p, max_new_tokens=24) for p in prompts]
        eng.step()
        eng.step()
        eng.abort_request(ids[0])
        eng.abort_request(ids[2])
        if compact:
            n = eng.compact_cache()
            assert {b for r in eng.running for b in r.blocks} == set(range(1, n + 1))
        drain(eng)
        return [eng.finished[i].output for i in ids]

    assert run(True) == run(False)
