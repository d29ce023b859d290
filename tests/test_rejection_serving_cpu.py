"""Sampled draft chains verified by rejection, through the engine and its sampler (CPU)."""
import dataclasses
from types import SimpleNamespace

import pytest
import torch

from phung5_b200 import ops
from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, preset
from phung5_b200.engine import engine as E
from phung5_b200.engine.oracle import SamplingParams
from phung5_b200.engine.sampling import seeded_coins, target_probs
from phung5_b200.models.llama import pack_weights
from phung5_b200.models.reference import RefModel
from phung5_b200.weights.init import random_weights


def _sampler(R, D, V, temps=None, top_k=0, top_p=1.0):
    """A _DraftSampler over a stand-in engine with whole vocabularies."""
    temps = torch.full((R,), 0.8) if temps is None else temps
    vocab = SimpleNamespace(full=lambda x: x)
    eng = SimpleNamespace(D=D, vocab=vocab, dvocab=vocab, cfg=SimpleNamespace(model=SimpleNamespace(vocab=V)),
                          sample_tensors=lambda reqs: (temps, torch.full((R,), top_k, dtype=torch.int32), torch.full((R,), top_p),
                                                       torch.arange(R) + 5, None))
    return E._DraftSampler(eng, [None] * R, torch.arange(R) + 11)


def test_dense_distributions_are_formed_in_bounded_pieces(monkeypatch):
    """64 requests x 5 drafts of a large vocabulary: no call of the dense definition takes more than 2^23 probabilities,
    and the step is the one that the whole tensors give."""
    R, D, V = 64, 5, 32003
    g = torch.Generator().manual_seed(3)
    dl = [torch.randn(R, V, generator=g) * 2 for _ in range(D)]
    vl = torch.randn(R, D + 1, V, generator=g) * 2
    for d in range(D):
        vl[:, d] = 0.9 * dl[d] + 0.2 * vl[:, d]               # near enough that drafts are kept
    sizes = []

    def spy(logits, *args):
        sizes.append(logits.numel())
        return target_probs(logits, *args)
    monkeypatch.setattr(E, "target_probs", spy)
    s = _sampler(R, D, V, top_k=50, top_p=0.95)
    drafts = [s.draw(x)[1] for x in dl]
    tokens = torch.cat([torch.zeros(R, 1, dtype=torch.int64)] + drafts, 1)
    acc, bonus = s.verify(vl, tokens)
    assert max(sizes) <= 1 << 23
    par = (torch.full((R,), 0.8), torch.full((R,), 50), torch.full((R,), 0.95))
    q = torch.stack([target_probs(x, *par) for x in dl], 1)
    p = torch.stack([target_probs(vl[:, d], *par) for d in range(D + 1)], 1)
    ra, rb = ops.spec_verify_probs(p, q, tokens[:, 1:], seeded_coins(torch.arange(R) + 5, torch.arange(R) + 11, D + 2))
    assert torch.equal(acc, ra) and torch.equal(bonus, rb)
    n = (acc >= 0).sum(1)
    assert 0 < int(n.sum()) < R * D
    for d, x in enumerate(drafts):
        assert bool((q[:, d].gather(1, x) > 0).all())


def _engine(accept, num_draft=2, model=None, drafter=None, **kw):
    return E.LLMEngine(EngineConfig(model=model or preset("tiny"), spec=SpecConfig(mode="chain", num_draft=num_draft, accept=accept),
                                    draft=DraftConfig(kind="model", num_layers=1), cache=CacheConfig(page_size=16, num_pages=128), **kw),
                       device="cpu", dtype=torch.float32, max_context=256, drafter=drafter)


def test_chains_without_drafts():
    """num_draft 0 emits one token a step, drawn from the target's distribution, under every accept rule."""
    eng = _engine("rejection", num_draft=0)
    outs = eng.generate([[1, 2, 3], [4, 5]], SamplingParams(max_new_tokens=5, temperature=0.8, seed=1))
    assert [len(o) for o in outs] == [5, 5] and all(a == 0 for r in eng.reqs.values() for a in r.accepted)
    again = _engine("rejection", num_draft=0).generate([[1, 2, 3], [4, 5]], SamplingParams(max_new_tokens=5, temperature=0.8, seed=1))
    assert again == outs


@pytest.mark.parametrize("accept", ["reject", "Rejection", "", "greedy"])
def test_unknown_accept_rules_are_refused(accept):
    with pytest.raises(ValueError, match="accept"):
        _engine(accept)


def test_accept_is_not_read_without_speculation():
    cfg = EngineConfig(model=preset("tiny"), spec=SpecConfig(enabled=False, accept="none"), cache=CacheConfig(page_size=16, num_pages=64))
    eng = E.LLMEngine(cfg, device="cpu", dtype=torch.float32, max_context=256)
    assert len(eng.generate([[1, 2]], SamplingParams(max_new_tokens=3))[0]) == 3


def test_rejection_needs_a_drafter_of_the_targets_vocabulary():
    """Refused when the engine is built, not in the middle of a step."""
    cfg = preset("tiny", num_layers=1, vocab=320)
    small = preset("tiny", num_layers=1, vocab=256)
    drafter = pack_weights(small, random_weights(small, seed=2, std=0.05), "cpu", dtype=torch.float32)
    with pytest.raises(ValueError, match="vocabulary"):
        _engine("rejection", model=cfg, drafter=drafter)
    same = pack_weights(cfg, random_weights(cfg, seed=2, std=0.05), "cpu", dtype=torch.float32)
    out = _engine("rejection", model=cfg, drafter=same).generate([[1, 2, 3]], SamplingParams(max_new_tokens=6, temperature=0.7, seed=2))
    assert len(out[0]) == 6


def test_the_drafts_of_a_chain_are_drawn_independently():
    """The second token after the root given the first, over 4000 seeds, against the target's distribution: drafts that
    share a coin would make it follow from the first. A frequency of n draws is off by more than 4.5 standard deviations (of
    at most 0.5 / sqrt(n)) about once in 10^5; some 300 frequencies are looked at."""
    cfg = dataclasses.replace(preset("tiny"), name="eight-tokens", num_layers=1, hidden=64, num_heads=2, num_kv_heads=2, head_dim=32,
                              ffn=96, vocab=8)
    w = random_weights(cfg, seed=7, std=0.3)
    g = torch.Generator().manual_seed(4)
    near = {k: v + 0.05 * torch.randn(v.shape, generator=g) if v.dim() == 2 else v for k, v in w.items()}
    pack = lambda x: pack_weights(cfg, x, "cpu", dtype=torch.float32)  # noqa: E731
    prompt, n = [3, 1, 4, 1, 5], 4000
    eng = E.LLMEngine(EngineConfig(model=cfg, spec=SpecConfig(mode="chain", num_draft=2, accept="rejection"), max_running=1024,
                                   draft=DraftConfig(kind="model", num_layers=1), cache=CacheConfig(page_size=16, num_pages=4096)),
                      device="cpu", dtype=torch.float32, max_context=256, target=pack(w), drafter=pack(near))
    rids = [eng.add_request(prompt, SamplingParams(max_new_tokens=3, temperature=1.0, seed=s)) for s in range(n)]
    while eng.has_work():
        eng.step()
    outs = [eng.reqs[r].out for r in rids]
    first = [eng.reqs[r].accepted[0] for r in rids]
    assert sum(a == 2 for a in first) > n // 4 and first.count(0) > n // 50       # both drafts kept, and rejections
    ref, seen = RefModel(cfg, w), 0
    for a in range(8):
        for b in range(8):
            group = [o[2] for o in outs if o[:2] == [a, b]]
            if len(group) < 100:
                continue
            logits, _ = ref.forward(torch.tensor(prompt + [a, b]), torch.arange(7), ref.new_cache())
            p = target_probs(logits[-1:], torch.ones(1), torch.zeros(1, dtype=torch.int64), torch.ones(1))[0]
            freq = torch.bincount(torch.tensor(group), minlength=8) / len(group)
            assert (freq - p).abs().max() < 4.5 * 0.5 / len(group) ** 0.5
            seen += 1
    assert seen >= 8
