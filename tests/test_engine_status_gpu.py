"""Errors that kernels report in the device's status word end the engine's step (the word is written from the host)."""
import pytest
import torch

from phung5_b200 import ops
from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, preset
from phung5_b200.engine.engine import LLMEngine
from phung5_b200.engine.oracle import SamplingParams

pytestmark = pytest.mark.gpu
PROMPTS = [[1, 2, 3] * 30, [5, 6, 7] * 50, [9, 8]]


def _engine(case):
    if case == "hybrid":
        cfg = EngineConfig(model=preset("hybrid-gdn-small", num_layers=4, gdn_prefill="chunked"), spec=SpecConfig(mode="chain", num_draft=3),
                           draft=DraftConfig(kind="model", num_layers=1), cache=CacheConfig(num_pages=128, max_seqs=8))
    else:
        cfg = EngineConfig(model=preset("small-bf16"), spec=SpecConfig(enabled=case != "decode", mode="chain", num_draft=3),
                           draft=DraftConfig(kind="eagle"), cache=CacheConfig(num_pages=128))
    return LLMEngine(cfg, device="cuda", max_context=2048)


@pytest.mark.parametrize("case", ["hybrid", "graph", "decode"])
def test_a_reported_error_ends_the_step(case):
    sp = SamplingParams(max_new_tokens=12)
    eng = _engine(case)
    ref = eng.generate(PROMPTS, sp)
    if case == "graph":
        assert eng.stats["graph_replays"] > 0
    for steps in (0, 2):
        rids = [eng.add_request(p, sp) for p in PROMPTS]
        for _ in range(steps):
            eng.step()
        ops.status_tensor("cuda")[0] = 8
        with pytest.raises(RuntimeError, match="outside its buffer"):
            eng.step()
        assert not eng.has_work() and all(eng.reqs[r].finish_reason == "abort" for r in rids)
        assert eng.pool.alloc.available() == 127 and not eng.pool.prefix.table
        assert int(ops.status_tensor("cuda")[0]) == 0
    assert eng.generate(PROMPTS, sp) == ref
