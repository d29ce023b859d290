"""Gated delta rule in chunks where a value is not finite or overflows, on the GPU: the result is the recurrence's."""
import math

import pytest
import torch

from phung5_b200 import ops
from phung5_b200.ops import gdn as G

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_BF16 = 2.0 ** -8      # a bf16 rounding is off by at most half a step: eps / 2 relative to the value


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status()


def _inputs(lens, hk, hv, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t, r = sum(lens), len(lens)
    q, k, v = (torch.randn(t, n, 128, generator=gen, device=DEV).bfloat16() for n in (hk, hk, hv))
    return dict(q=q, k=k, v=v, g=-torch.rand(t, hv, generator=gen, device=DEV) * 0.2,
                beta=torch.rand(t, hv, generator=gen, device=DEV) * 0.9 + 0.05,
                state=torch.randn(r + 1, hv, 128, 128, generator=gen, device=DEV) * 0.2,
                tok_start=torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV),
                slot=torch.arange(r, dtype=torch.int32, device=DEV).flip(0), scale=1 / math.sqrt(128))


def _definition(a):
    """Token by token in 64 bits, on the CPU."""
    b = {k: x.cpu() if isinstance(x, torch.Tensor) else x for k, x in a.items()}
    rep = b["v"].shape[1] // b["q"].shape[1]
    unit = lambda x: (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(rep, 1)  # noqa: E731
    q, k, v = unit(b["q"].double()) * b["scale"], unit(b["k"].double()), b["v"].double()
    pool, out = b["state"].double(), torch.zeros(b["v"].shape, dtype=torch.float64)
    ts = b["tok_start"].tolist()
    for r, s in enumerate(b["slot"].tolist()):
        S = pool[s].clone()
        for i in range(ts[r], ts[r + 1]):
            S = S * b["g"][i].double().exp()[:, None, None]
            vp = b["beta"][i].double()[:, None] * (v[i] - torch.einsum("hij,hi->hj", S, k[i]))
            S = S + k[i][:, :, None] * vp[:, None, :]
            out[i] = torch.einsum("hij,hi->hj", S, q[i])
        pool[s] = S
    return out.to(DEV), pool.to(DEV)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("token", [9, 95, 199])
def test_gdn_chunked_not_finite_reaches_no_earlier_token(what, value, token):
    """One value that is not finite, in the first, the second and the request's short last chunk: exactly the outputs and
    elements of the state that the definition makes not finite are so, and the others are what they are without it."""
    lens = [200, 70]
    a = _inputs(lens, 2, 4, seed=token)
    if what == "state":
        a["state"][int(a["slot"][0]), 1, 3, 5] = value
    else:
        a[what][(token, 1) + ((5,) if what in ("q", "k", "v") else ())] = value
    out, pool = _definition(a)
    start = a["state"].clone()
    got = G.gdn_chunked(**a)
    torch.cuda.synchronize()
    fin = out.isfinite()
    if what != "state":
        assert bool(fin[:token].all()) and not bool(fin.all())
    assert torch.equal(got.isfinite(), fin)
    # out: one bf16 rounding on a sum of 128 products in fp32 or of bf16 pieces (2^-16 an operand, five products in a row),
    # against the largest magnitude about
    big = out[fin].abs().max()
    assert bool(((got.double() - out).abs()[fin] <= HALF_BF16 * out.abs()[fin] + 2.0 ** -13 * big).all())
    fin = pool.isfinite()
    assert torch.equal(a["state"].isfinite(), fin)
    assert bool(((a["state"].double() - pool).abs()[fin] <= 2.0 ** -14 * pool[fin].abs().max()).all())
    assert torch.equal(a["state"][2], start[2])
    again = G.gdn_chunked(**{**a, "state": start})
    assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(got))


@pytest.mark.parametrize("what,value", [("k", 2.0 ** 100), ("q", 2.0 ** 100), ("v", 2.0 ** 125)])
def test_gdn_chunked_overflows_as_the_recurrence_does(what, value):
    """Finite inputs whose squares or sums pass fp32's range: the chunk form gives what the token-by-token form gives."""
    a = _inputs([200, 70], 2, 4, seed=8)
    a[what][70] = value * torch.sign(a[what][70])
    b = {**a, "state": a["state"].clone()}
    ref, _ = G.gdn_recurrent(**b, write_state=True, stash=False)
    got = G.gdn_chunked(**a)
    fin = ref.isfinite()
    assert bool(fin[:70].all())
    assert torch.equal(got.isfinite(), fin)
    # each is off by half a step and by its sums' rounding (2^-13 of the largest magnitude about)
    for rows in (slice(0, 70), slice(70, 200), slice(200, 270)):
        x, y = got[rows].double(), ref[rows].double()
        x, y = x[fin[rows]], y[fin[rows]]
        if x.numel():
            assert bool(((x - y).abs() <= 2 * HALF_BF16 * y.abs() + 2.0 ** -12 * y.abs().max()).all())
    fin = b["state"].isfinite()
    assert torch.equal(a["state"].isfinite(), fin)


@pytest.mark.parametrize("which", ["q", "k", "v", "out"])
def test_gdn_chunked_long_run_off_the_boundaries(which):
    """A long run with one operand off 16-byte boundaries goes token by token: the same recurrence."""
    a = _inputs([700, 300], 2, 4, seed=3)
    out, pool = _definition(a)
    shift = lambda x: torch.empty(x.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(x.shape)  # noqa: E731
    if which == "out":
        got = G.gdn_chunked(**a, out=shift(a["v"]))
    else:
        got = G.gdn_chunked(**{**a, which: shift(a[which]).copy_(a[which])})
    # one bf16 rounding; sums of 128 products in fp32 over a memory of some ten tokens stay below 2^-13 of the largest value
    assert bool(((got.double() - out).abs() <= HALF_BF16 * out.abs() + 2.0 ** -13 * out.abs().max()).all())
    assert bool(((a["state"].double() - pool).abs() <= 2.0 ** -14 * pool.abs().max()).all())
