"""Models with per-head q/k norms, chunked prompt passes of hybrid models and sampled draft chains verified by rejection,
through the engine (CPU, fp32)."""
import dataclasses

import pytest
import torch

from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, load_engine_config, preset
from phung5_b200.engine.engine import LLMEngine
from phung5_b200.engine.oracle import SamplingParams, greedy_generate
from phung5_b200.engine.sampling import target_probs
from phung5_b200.models.llama import pack_weights
from phung5_b200.models.reference import RefModel
from phung5_b200.weights.init import random_weights
from phung5_b200.weights.loader import load_model, save_checkpoint


def _normed_weights(cfg, seed=3):
    w = random_weights(cfg, seed=seed, std=0.05)
    g = torch.Generator().manual_seed(seed)
    for k in w:
        if k.endswith("q_norm.weight") or k.endswith("k_norm.weight"):
            w[k] = 1 + 0.3 * torch.randn(w[k].shape, generator=g)
    return w


def _engine(cfg, w=None, drafter=None, temperature_mode="exact", num_draft=3, **kw):
    ecfg = EngineConfig(model=cfg, spec=SpecConfig(mode="chain", num_draft=num_draft, accept=temperature_mode),
                        draft=DraftConfig(kind="model", num_layers=1), cache=CacheConfig(page_size=16, num_pages=512, max_seqs=64), **kw)
    t = None if w is None else pack_weights(cfg, w, "cpu", dtype=torch.float32)
    return LLMEngine(ecfg, device="cpu", dtype=torch.float32, max_context=512, target=t, drafter=drafter)


def test_qk_norm_model_equals_the_oracle(tmp_path):
    cfg = preset("tiny", num_layers=2, qk_norm=True)
    w = _normed_weights(cfg)
    prompt = torch.randint(0, cfg.vocab, (21,), generator=torch.Generator().manual_seed(1)).tolist()
    ref = greedy_generate(RefModel(cfg, w), prompt, 10)
    plain = {k: v for k, v in w.items() if "q_norm" not in k and "k_norm" not in k}
    assert greedy_generate(RefModel(cfg, plain), prompt, 10) != ref          # the norms matter here
    assert _engine(cfg, w).generate([prompt], SamplingParams(max_new_tokens=10)) == [ref]
    # a checkpoint that holds the norms' weights is served with them
    save_checkpoint(w, cfg, str(tmp_path), shards=2)
    mc, packed = load_model(str(tmp_path), "cpu")
    assert mc.qk_norm and torch.equal(packed.layers[1].k_norm.float(), w["model.layers.1.self_attn.k_norm.weight"].bfloat16().float())


def test_hybrid_chunked_prefill_and_qk_norm_equal_the_recurrent_path():
    g = torch.Generator().manual_seed(11)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (37, 70, 5)]
    outs = []
    for prefill in ("recurrent", "chunked"):
        cfg = preset("tiny-hybrid", qk_norm=True, gdn_prefill=prefill)
        eng = _engine(cfg)
        assert all(x is None or x.gdn.chunked == (prefill == "chunked") for x in eng.target.gdn_layers)
        assert all(x.q_norm is not None for x in eng.tw.layers)
        outs.append(eng.generate(prompts, SamplingParams(max_new_tokens=9)))
    assert outs[0] == outs[1]
    with pytest.raises(ValueError, match="gdn_prefill"):
        _engine(preset("tiny-hybrid", gdn_prefill="scan"))


def test_rejection_is_for_chains():
    with pytest.raises(ValueError, match="chain"):
        LLMEngine(EngineConfig(model=preset("tiny"), spec=SpecConfig(mode="tree", accept="rejection"), draft=DraftConfig(kind="model"),
                               cache=CacheConfig(page_size=16, num_pages=64)), device="cpu", dtype=torch.float32)
    cfg = load_engine_config(overrides={"model": "tiny", "spec.accept": "rejection", "spec.mode": "chain"})
    assert cfg.spec.accept == "rejection"


def test_rejection_with_the_target_as_its_own_drafter_keeps_every_draft():
    cfg = preset("tiny", num_layers=2, vocab=300)
    w = random_weights(cfg, seed=5, std=0.05)
    packed = pack_weights(cfg, w, "cpu", dtype=torch.float32)
    eng = _engine(cfg, w, drafter=packed, temperature_mode="rejection")
    outs = eng.generate([[1, 2, 3, 4], [9, 8, 7]], SamplingParams(max_new_tokens=17, temperature=0.9, top_k=0, seed=4))
    acc = [a for r in eng.reqs.values() for a in r.accepted]
    assert all(len(o) == 17 for o in outs) and len(acc) > 4 and sum(acc) >= 3 * len(acc) - 1     # p = q up to rounding
    greedy = _engine(cfg, w, drafter=packed, temperature_mode="rejection").generate([[1, 2, 3, 4]], SamplingParams(max_new_tokens=9))
    assert greedy[0] == greedy_generate(RefModel(cfg, w), [1, 2, 3, 4], 9)


def test_rejection_follows_the_targets_distribution():
    """The first token after the root, over 2000 seeds, against the target's distribution given that root. A frequency of
    n draws is off by more than 4.5 standard deviations (of at most 0.5 / sqrt(n)) about once in 10^5."""
    cfg = dataclasses.replace(preset("tiny"), name="eight-tokens", num_layers=1, hidden=64, num_heads=2, num_kv_heads=2, head_dim=32, ffn=96, vocab=8)
    w = random_weights(cfg, seed=7, std=0.3)
    prompt, n = [3, 1, 4, 1, 5], 2000
    eng = _engine(cfg, w, temperature_mode="rejection", num_draft=2, max_running=512)
    rids = [eng.add_request(prompt, SamplingParams(max_new_tokens=4, temperature=1.0, seed=s)) for s in range(n)]
    while eng.has_work():
        eng.step()
    outs = [eng.reqs[r].out for r in rids]
    acc = [a for r in rids for a in eng.reqs[r].accepted]
    assert 0 in acc and 2 in acc                    # drafts are both kept and rejected
    ref = RefModel(cfg, w)
    for root in range(8):
        group = [o[1] for o in outs if o[0] == root]
        if len(group) < 150:
            continue
        logits, _ = ref.forward(torch.tensor(prompt + [root]), torch.arange(6), ref.new_cache())
        p = target_probs(logits[-1:], torch.ones(1), torch.zeros(1, dtype=torch.int64), torch.ones(1))[0]
        freq = torch.bincount(torch.tensor(group), minlength=8) / len(group)
        assert (freq - p).abs().max() < 4.5 * 0.5 / len(group) ** 0.5


def test_hybrid_rejection_runs_with_everything_on():
    """Chunked prompt passes, normed heads and sampled chains together: reproducible, and mixed with greedy requests that
    emit what they emit alone."""
    cfg = preset("tiny-hybrid", qk_norm=True, gdn_prefill="chunked")
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (40, 21)]

    def run(temps):
        eng = _engine(cfg, temperature_mode="rejection")
        rids = [eng.add_request(p, SamplingParams(max_new_tokens=8, temperature=t, top_k=50, top_p=0.9, seed=6)) for p, t in zip(prompts, temps)]
        while eng.has_work():
            eng.step()
        assert eng.stats["spec_steps"] > 0 and sorted(eng.gdn_pool.free) == list(range(64))
        return [eng.reqs[r].out for r in rids]

    a, b, mixed, greedy = run((0.8, 0.8)), run((0.8, 0.8)), run((0.8, 0.0)), run((0.0, 0.0))
    assert a == b and mixed == [a[0], greedy[1]] and a != greedy


def test_bounds_checks_pass_on_a_whole_run():
    """Every index that the engine hands to these operators passes the bounds-check mode, and it changes no token."""
    from phung5_b200.ops import check
    cfg = preset("tiny-hybrid", qk_norm=True, gdn_prefill="chunked")
    prompts, sp = [[1, 2, 3, 4, 5] * 6, [7, 8, 9]], SamplingParams(max_new_tokens=6, temperature=0.8, top_k=20, seed=3)
    ref = _engine(cfg, temperature_mode="rejection").generate(prompts, sp)
    with check.bounds_checks():
        before = check.CHECKS[0]
        assert _engine(cfg, temperature_mode="rejection").generate(prompts, sp) == ref
        assert check.CHECKS[0] > before
