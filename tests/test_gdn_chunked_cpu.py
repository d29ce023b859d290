"""Arguments of the chunked gated delta rule (CPU)."""
import pytest
import torch

from phung5_b200.ops import gdn as G


def _inputs(t=6, hk=1, hv=2):
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(t, n, 128, generator=gen) for n in (hk, hk, hv))
    return dict(q=q, k=k, v=v, g=-torch.rand(t, hv, generator=gen), beta=torch.rand(t, hv, generator=gen),
                state=torch.zeros(1, hv, 128, 128), tok_start=torch.tensor([0, t], dtype=torch.int32),
                slot=torch.zeros(1, dtype=torch.int32), scale=0.1)


def test_gdn_chunked_refuses_an_output_in_an_inputs_memory():
    """A request that is taken again reads its inputs after outputs were written: they may not share memory."""
    a = _inputs()
    ref = G.gdn_chunked(**{**a, "state": a["state"].clone()})
    buf = torch.zeros(2, 6, 2, 128)
    for x in ("v", "q"):
        b = {**a, "state": a["state"].clone()}
        if x == "v":
            out = b["v"]
        else:
            wide = buf.view(12, 2, 128)
            b["q"] = wide[5:11, :1].copy_(a["q"])
            out = wide[:6]
        with pytest.raises(ValueError, match="shares memory"):
            G.gdn_chunked(**b, out=out)
        assert torch.equal(b["state"], a["state"])
    b = {**a, "v": buf[0].copy_(a["v"]), "state": a["state"].clone()}        # neighbours in one allocation are fine
    assert torch.equal(G.gdn_chunked(**b, out=buf[1]), ref)
