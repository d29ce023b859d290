"""Sampled draft chains verified by rejection, through the engine's sampler, on the GPU."""
import pytest
import torch

from phung5_b200 import ops
from test_rejection_serving_cpu import _sampler

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status()


def test_rejection_step_holds_its_results_and_one_piece():
    """256 requests x 2 drafts x 128256 tokens: beside the two dense results a step holds at most 0.5 GiB, the piece of
    2^23 probabilities whose sorted values, indices and sums take up to 64 bytes each."""
    R, D, V = 256, 2, 128256
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = torch.randn(R, D + 1, V, generator=g, device=DEV)
    with torch.device(DEV):
        s = _sampler(R, D, V, top_k=50, top_p=0.95)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    tokens = torch.zeros(R, D + 1, dtype=torch.int64, device=DEV)
    for d in range(D):
        tokens[:, d + 1:d + 2] = s.draw(logits[:, d])[1]
    acc, bonus = s.verify(logits, tokens)
    torch.cuda.synchronize()
    held = torch.cuda.max_memory_allocated() - base
    results = 4 * R * V * (D + D + 1)
    assert held <= results + 64 * 2 ** 23 + 2 ** 20, held
    assert bool((acc >= 0).all())                    # the drafts' distributions are the target's own
    assert bool(((bonus >= 0) & (bonus < V)).all())
