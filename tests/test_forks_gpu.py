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


def rows(eng, r, upto):
    """Request r's cached keys and values of every layer, [layers, 2, upto, heads, D] as they read back."""
    at = torch.arange(upto, device="cuda")
    slots = torch.tensor(r.blocks, device="cuda")[at // 64] * 64 + at % 64
    out = []
    for k, v in eng.caches:
        if k.dtype == torch.uint8:
            out.append(torch.stack(ops.kv_fp4_read(k, v, slots, eng.cfg.model.head_dim)))
        else:
            out.append(torch.stack([c[slots // 64, :, slots % 64] for c in (k, v)]))
    return torch.stack(out)


@pytest.mark.parametrize("kv", ["nvfp4", "bf16"])
@pytest.mark.parametrize("length", [100, 128, 333])
def test_a_fork_holds_its_parents_rows_bit_for_bit(kv, length):
    eng = engine(kv=kv)
    rng = np.random.default_rng(length)
    a = eng.add_request(rng.integers(0, 1024, length), max_new_tokens=40)
    for _ in range(4):
        eng.step()
    parent = eng.running[0]
    b = eng.fork_request(a, [3, 1, 4], max_new_tokens=10)
    child, n = eng.waiting[0], parent.committed
    assert child.prefilled == n and (n % 64 == 0 or child.blocks[-1] not in parent.blocks)
    want = rows(eng, parent, n).clone()
    assert want.float().abs().sum() > 0
    assert torch.equal(rows(eng, child, n), want)
    while not any(r.rid == b for r in eng.running):
        eng.step()
    for _ in range(3):
        eng.step()
    # both have written on: neither has touched what the other holds
    assert torch.equal(rows(eng, child, n), want) and torch.equal(rows(eng, parent, n), want)
    eng.compact_cache()
    assert torch.equal(rows(eng, child, n), want) and torch.equal(rows(eng, parent, n), want)


def test_every_fork_continues_as_a_fresh_request_would(monkeypatch):
    """In batch-invariant mode a row of the 4-bit attention depends neither on the other rows nor on the table's width,
    so a prompt's tokens get the bits that decode steps gave them."""
    monkeypatch.setenv("SH_BATCH_INVARIANT", "1")
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, 1024, n) for n in (100, 640, 333)]
    eng = engine()
    free = eng.pool.free
    ids = [eng.add_request(p, max_new_tokens=30) for p in prompts]
    for _ in range(5):
        eng.step()
    outs = [list(r.output) for r in eng.running]
    kids = [(i, x, eng.fork_request(ids[i], x, max_new_tokens=10)) for i in range(3) for x in ([], [3, 1, 4])]
    while eng.has_work():
        eng.step()
    assert eng.pool.free == free
    for i, x, kid in kids:
        fresh = engine().generate([np.concatenate([prompts[i], outs[i], x]).astype(np.int64)], 10)[0]
        assert eng.finished[kid].output == fresh, (i, x)
        if not x:
            assert fresh == eng.finished[ids[i]].output[len(outs[i]):len(outs[i]) + 10]
