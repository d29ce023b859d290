"""Errors that kernels report in the status word end the engine's step (CPU, with a stand-in for the word)."""
import pytest
import torch

from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, preset
from phung5_b200.engine.engine import LLMEngine
from phung5_b200.engine.oracle import SamplingParams


class _Word:
    """A status word that holds an error from its `at`-th reading on, until it is raised."""

    def __init__(self, at):
        self.at, self.reads, self.fetched = at, 0, False

    def fetch(self):
        self.fetched = True
        return 0

    def check(self):
        assert self.fetched            # copied before the step waited for the device
        self.fetched = False
        self.reads += 1
        if self.reads == self.at:
            raise RuntimeError("kernel status: planted")


def _engine(model="tiny", spec=True, **kw):
    return LLMEngine(EngineConfig(model=preset(model), spec=SpecConfig(enabled=spec, mode="chain", num_draft=2),
                                  draft=DraftConfig(kind="model", num_layers=1), cache=CacheConfig(page_size=16, num_pages=128, max_seqs=8), **kw),
                     device="cpu", dtype=torch.float32, max_context=256)


PROMPTS = [[1, 2, 3] * 7, [5, 6, 7] * 12, [9, 8]]


@pytest.mark.parametrize("at", [1, 2, 4])
@pytest.mark.parametrize("model,spec", [("tiny", True), ("tiny", False), ("tiny-hybrid", True)])
def test_a_reported_error_ends_the_step(model, spec, at):
    """The first reading is the prompt pass's, the others the next steps'. Nothing of the failed step is emitted, its
    requests are dropped with their pages, states and cached prefixes, and the engine serves on."""
    sp = SamplingParams(max_new_tokens=9)
    ref = _engine(model, spec).generate(PROMPTS, sp)
    eng = _engine(model, spec)
    eng._status = _Word(at)
    rids = [eng.add_request(p, sp) for p in PROMPTS]
    emitted = {r: [] for r in rids}
    with pytest.raises(RuntimeError, match="planted"):
        while eng.has_work():
            for o in eng.step():
                emitted[o.rid] += o.new_tokens
    for r, want in zip(rids, ref):
        q = eng.reqs[r]
        assert q.finished and q.finish_reason in ("abort", "length") and not q.pages
        assert q.out == want[:len(q.out)] and emitted[r] == q.out[:len(emitted[r])]
    assert not eng.has_work() and not eng.running and not eng.waiting
    assert eng.pool.alloc.available() == 127 and not eng.pool.prefix.table and not eng.pool.prefix.lru
    if model == "tiny-hybrid":
        assert sorted(eng.gdn_pool.free) == list(range(8))
    assert eng.generate(PROMPTS, sp) == ref


def test_requests_that_had_not_started_stay_queued():
    sp = SamplingParams(max_new_tokens=6)
    ref = _engine().generate(PROMPTS, sp)
    eng = _engine(max_running=1)
    eng._status = _Word(2)
    rids = [eng.add_request(p, sp) for p in PROMPTS]
    with pytest.raises(RuntimeError, match="planted"):
        while eng.has_work():
            eng.step()
    assert [eng.reqs[r].finished for r in rids] == [True, False, False]
    while eng.has_work():
        eng.step()
    assert [eng.reqs[r].out for r in rids[1:]] == ref[1:]
