"""Graph captures, forks and page copies of the engine on the GPU."""
import dataclasses

import numpy as np
import pytest
import torch

from vllm_suffix_hybrid_b200 import ops
from vllm_suffix_hybrid_b200.engine.config import CacheConfig, EngineConfig, SpecConfig, llama3_8b_config, shrink
from vllm_suffix_hybrid_b200.engine.llm import LLMEngine

pytestmark = pytest.mark.gpu


def engine(method="none", kv="nvfp4", seqs=4, graphs=True, layers=3, budget=4096):
    m = dataclasses.replace(shrink(llama3_8b_config(), layers=layers, hidden=256, vocab=1024), kv_format=kv)
    return LLMEngine(EngineConfig(model=m, spec=SpecConfig(method=method, k=3), cache=CacheConfig(max_model_len=2048),
                                  max_num_seqs=seqs, device="cuda", cuda_graphs=graphs, max_prefill_tokens=budget))


def test_all_captures_warm_up_on_one_stream(monkeypatch):
    """Attention keeps its partials by stream for good: a new stream for each graph would keep a set each."""
    eng = engine(seqs=8)
    streams, real, main = set(), eng.runner._decode_body, torch.cuda.current_stream().cuda_stream

    def spy(*args):
        if not torch.cuda.is_current_stream_capturing():
            streams.add(torch.cuda.current_stream().cuda_stream)
        return real(*args)

    monkeypatch.setattr(eng.runner, "_decode_body", spy)
    rng = np.random.default_rng(5)
    for n in (1, 2, 4, 8):
        eng.generate([rng.integers(0, 1024, 40) for _ in range(n)], 4)
    assert len(eng.runner.graphs) >= 3 and len(streams) == 1 and main not in streams
