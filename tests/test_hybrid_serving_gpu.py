"""Hybrid models with normed heads, chunked prompt passes and sampled draft chains verified by rejection, on the GPU: the
kernels run one after the other as the engine uses them."""
import pytest
import torch

from phung5_b200 import ops
from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, preset
from phung5_b200.engine.attn_meta import build_items, make_meta, pack_work
from phung5_b200.engine.engine import LLMEngine
from phung5_b200.engine.oracle import SamplingParams
from phung5_b200.models.hybrid import GdnBatch, random_hybrid
from phung5_b200.models.llama import ForwardBatch, random_packed_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status()


def _hybrid(prefill, accept="exact"):
    cfg = preset("hybrid-gdn-small", num_layers=4, qk_norm=True, gdn_prefill=prefill)
    target, gdn = random_hybrid(cfg, DEV, seed=1, std=0.05)
    gen = torch.Generator(device=DEV).manual_seed(5)
    for lw in target.layers:
        lw.q_norm = (1 + 0.2 * torch.randn(128, generator=gen, device=DEV)).bfloat16()
        lw.k_norm = (1 + 0.2 * torch.randn(128, generator=gen, device=DEV)).bfloat16()
    ecfg = EngineConfig(model=cfg, spec=SpecConfig(mode="chain", num_draft=3, accept=accept), draft=DraftConfig(kind="model", num_layers=1),
                        cache=CacheConfig(num_pages=128, max_seqs=8))
    return LLMEngine(ecfg, device=DEV, target=(target, gdn), max_context=2048)


def _prefill(eng, prompts):
    lens = [len(p) for p in prompts]
    pages = [eng.pool.prefix.alloc_pages((n + 63) // 64) for n in lens]
    meta = make_meta(pages, [0] * len(lens), lens, None, True, DEV)
    g = eng.target.hq // eng.target.hkv
    _, p2 = build_items(meta, g)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    fb = ForwardBatch(tokens=torch.tensor(sum(prompts, []), device=DEV),
                      positions=torch.cat([torch.arange(n, dtype=torch.int32, device=DEV) for n in lens]),
                      slots=torch.tensor([pg[i // 64] * 64 + i % 64 for pg, n in zip(pages, lens) for i in range(n)], device=DEV),
                      meta=meta, work2=pack_work(p2, g, DEV))
    fb.gdn = GdnBatch(torch.tensor(starts, dtype=torch.int32, device=DEV),
                      torch.tensor([eng.gdn_pool.alloc() for _ in lens], dtype=torch.int32, device=DEV), "prefill")
    logits, _ = eng.target.forward(fb)
    return logits.float(), eng.gdn_pool.state.clone()


def test_chunked_prompt_pass_equals_the_recurrent_one():
    """The first GDN layer sees the same inputs either way, so its states agree to fp32; further on the two paths differ by
    single bf16 roundings (2^-8 of a value) in the outputs of three GDN layers, each normed again before its projection:
    below 2^-5 of the logits' norm."""
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 32000, (n,), generator=g).tolist() for n in (333, 64, 5, 700)]
    (la, sa), (lb, sb) = _prefill(_hybrid("recurrent"), prompts), _prefill(_hybrid("chunked"), prompts)
    assert ((sa[0] - sb[0]).norm() / sa[0].norm()).item() < 2e-5
    assert ((sa - sb).norm() / sa.norm()).item() < 2.0 ** -5
    assert ((la - lb).norm() / la.norm()).item() < 2.0 ** -5


def test_hybrid_rejection_with_everything_on():
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 32000, (n,), generator=g).tolist() for n in (150, 40, 9)]

    def run(temps):
        eng = _hybrid("chunked", "rejection")
        rids = [eng.add_request(p, SamplingParams(max_new_tokens=12, temperature=t, top_k=0, top_p=0.95, seed=8)) for p, t in zip(prompts, temps)]
        while eng.has_work():
            eng.step()
        assert eng.stats["spec_steps"] > 0 and len(eng.gdn_pool.free) == 8
        outs = [eng.reqs[r].out for r in rids]
        assert all(len(o) == 12 and all(0 <= t < 32000 for t in o) for o in outs)
        return outs

    a = run((0.7, 0.7, 0.0))
    assert a == run((0.7, 0.7, 0.0))             # seeded: the same tokens again
    assert a[0] != run((0.0, 0.7, 0.0))[0]


def test_rejection_with_the_target_as_its_own_drafter():
    """p and q differ by the rounding of two forwards of other shapes: nearly every draft is kept."""
    cfg = preset("small-bf16", qk_norm=True)
    w = random_packed_weights(cfg, DEV, seed=2, std=0.05)
    eng = LLMEngine(EngineConfig(model=cfg, spec=SpecConfig(mode="chain", num_draft=4, accept="rejection"),
                                 draft=DraftConfig(kind="model", num_layers=2), cache=CacheConfig(num_pages=128)),
                    device=DEV, target=w, drafter=w, max_context=1024)
    prompts = [torch.randint(0, 8192, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (50, 90)]
    outs = eng.generate(prompts, SamplingParams(max_new_tokens=41, temperature=1.0, top_k=0, seed=3))
    acc = [a for r in eng.reqs.values() for a in r.accepted]
    assert all(len(o) == 41 for o in outs) and sum(acc) >= 3 * len(acc)
