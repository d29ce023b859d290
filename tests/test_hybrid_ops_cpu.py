"""Chunked gated delta rule, per-head q/k norm with rotation and cache write, verification of sampled draft chains:
their CPU definitions against independent 64-bit forms, their refusals and their bounds checks."""
import math

import pytest
import torch

from phung5_b200 import ops
from phung5_b200.engine.sampling import seeded_coins
from phung5_b200.ops import gdn as G
from phung5_b200.ops.check import BoundsError, bounds_checks


# ---- gated delta rule ------------------------------------------------------------------------------------------

def _gdn_inputs(lens, hk, hv, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    t = sum(lens) + extra
    ts = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    return dict(q=torch.randn(t, hk, 128, generator=g), k=torch.randn(t, hk, 128, generator=g),
                v=torch.randn(t, hv, 128, generator=g), g=-torch.rand(t, hv, generator=g),
                beta=torch.rand(t, hv, generator=g), state=torch.randn(len(lens) + 2, hv, 128, 128, generator=g) * 0.1,
                tok_start=ts, slot=torch.arange(len(lens), dtype=torch.int32) + 1, scale=1 / math.sqrt(128))


def test_gdn_chunked_definition_solves_the_chunk_equations():
    """(I + L) V' = beta (V - e^b K S0), O = e^b Q S0 + tril(Q K^T e^(b_i - b_j)) V', S1 = e^bC S0 + ..., solved in fp64
    for the whole run as one chunk."""
    a = _gdn_inputs([7], 1, 2)
    s0 = a["state"][1].double()
    out = G.gdn_chunked(**a)
    for h in range(2):
        q, k, v = a["q"][:, 0].double(), a["k"][:, 0].double(), a["v"][:, h].double()
        q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt() * a["scale"]
        k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
        b, beta = a["g"][:, h].double().cumsum(0), a["beta"][:, h].double()[:, None]
        decay = (b[:, None] - b[None, :]).exp()
        L = (beta * decay * (k @ k.T)).tril(-1)
        vp = torch.linalg.solve(torch.eye(7).double() + L, beta * (v - b.exp()[:, None] * (k @ s0[h])))
        o = b.exp()[:, None] * (q @ s0[h]) + (decay * (q @ k.T)).tril() @ vp
        s1 = b[-1].exp() * s0[h] + (k * (b[-1] - b).exp()[:, None]).T @ vp
        assert torch.allclose(out[:, h].double(), o, atol=1e-5)
        assert torch.allclose(a["state"][1, h].double(), s1, atol=1e-5)


def test_gdn_chunked_leaves_other_rows_and_slots():
    a = _gdn_inputs([3, 0, 2], 1, 1, extra=4)
    before = a["state"].clone()
    out = torch.full((9, 1, 128), 7.0)
    G.gdn_chunked(**a, out=out)
    assert (out[5:] == 7).all() and not (out[:5] == 7).any()
    assert torch.equal(a["state"][[0, 2, 4]], before[[0, 2, 4]])       # unused slots, and the request without tokens
    assert not torch.equal(a["state"][1], before[1]) and not torch.equal(a["state"][3], before[3])


def test_gdn_chunked_refusals():
    a = _gdn_inputs([3], 2, 4)
    for key, bad in (("k", a["k"][:, :1]), ("q", a["q"][..., :64]), ("v", a["v"][:2]), ("slot", torch.zeros(2, dtype=torch.int32)),
                     ("v", torch.randn(3, 3, 128))):
        with pytest.raises((ValueError, RuntimeError)):
            G.gdn_chunked(**{**a, key: bad})
    with bounds_checks():
        G.gdn_chunked(**a)
        with pytest.raises(BoundsError, match="slot"):
            G.gdn_chunked(**{**a, "slot": torch.tensor([3], dtype=torch.int32)})
        with pytest.raises(BoundsError, match="tok_start"):
            G.gdn_chunked(**{**a, "tok_start": torch.tensor([0, 4], dtype=torch.int32)})
        b = _gdn_inputs([2, 2], 1, 1)
        with pytest.raises(BoundsError, match="more than once"):
            G.gdn_chunked(**{**b, "slot": torch.tensor([1, 1], dtype=torch.int32)})
        with pytest.raises(BoundsError, match="decreases"):
            G.gdn_chunked(**{**b, "tok_start": torch.tensor([0, 4, 2], dtype=torch.int32)})


# ---- q/k norm + rotation + cache write -------------------------------------------------------------------------

def _qk_inputs(m=5, hq=4, hkv=2, d=16, rot=16, pages=3, ps=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    return dict(qkv=torch.randn(m, (hq + 2 * hkv) * d, generator=g), wq=1 + 0.3 * torch.randn(d, generator=g),
                wk=1 + 0.3 * torch.randn(d, generator=g), eps=1e-6, pos=torch.arange(m, dtype=torch.int32) + 3,
                slots=torch.tensor([0, 5, -1, 11, 7][:m]), cos_sin=ops.rope_table(32, rot, 1e4, "cpu"),
                k_cache=torch.zeros(pages, hkv, ps, d), v_cache=torch.zeros(pages, hkv, ps, d), hq=hq, hkv=hkv, d=d)


@pytest.mark.parametrize("rot", [16, 8, 2])
def test_qk_norm_is_norm_then_rope(rot):
    """Normed heads fed through rope_kv_write (whole rotation), the rest of a partially rotated head only normed."""
    a = _qk_inputs(rot=rot)
    q = ops.qk_norm_rope_kv_write(**a)
    x = a["qkv"].double().view(5, 8, 16)
    y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    yq, yk = y[:, :4] * a["wq"].double(), y[:, 4:6] * a["wk"].double()
    part = torch.cat([yq[..., :rot].reshape(5, -1), yk[..., :rot].reshape(5, -1), x[:, 6:, :rot].reshape(5, -1)], 1)
    kc, vc = torch.zeros(3, 2, 4, rot), torch.zeros(3, 2, 4, rot)
    qr = ops.rope_kv_write(part.float(), a["pos"], a["slots"], a["cos_sin"], kc, vc, 4, 2, rot)
    assert torch.allclose(q[..., :rot], qr, atol=1e-5)
    assert torch.allclose(q[..., rot:].double(), yq[..., rot:], atol=1e-5)
    assert torch.allclose(a["k_cache"][..., :rot], kc, atol=1e-5)
    for t, s in enumerate(a["slots"].tolist()):
        if s >= 0:
            assert torch.allclose(a["k_cache"][s // 4, :, s % 4, rot:].double(), yk[t, :, rot:], atol=1e-5)
            assert torch.equal(a["v_cache"][s // 4, :, s % 4], a["qkv"].view(5, 8, 16)[t, 6:])
    assert int((a["v_cache"].abs().sum(-1) > 0).sum()) == 4 * 2         # four rows with a slot, two heads


def test_qk_norm_refusals():
    a = _qk_inputs()
    for key, bad in (("qkv", a["qkv"][:, :-1]), ("wq", a["wq"][:8]), ("wk", torch.ones(17)),
                     ("cos_sin", ops.rope_table(32, 32, 1e4, "cpu"))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.qk_norm_rope_kv_write(**{**a, key: bad})
    with bounds_checks():
        ops.qk_norm_rope_kv_write(**a)
        with pytest.raises(BoundsError, match="slots"):
            ops.qk_norm_rope_kv_write(**{**a, "slots": torch.tensor([0, 12, 1, 2, 3])})
        with pytest.raises(BoundsError, match="more than once"):
            ops.qk_norm_rope_kv_write(**{**a, "slots": torch.tensor([3, 4, 3, -1, 0])})
        with pytest.raises(BoundsError, match="pos"):
            ops.qk_norm_rope_kv_write(**{**a, "pos": torch.tensor([0, 1, 2, 3, 32], dtype=torch.int32)})


# ---- verification of sampled draft chains ----------------------------------------------------------------------

def test_verify_emits_the_targets_distribution():
    """Over a fine grid of both coins and every draft (weighted by q), the first emitted token follows p."""
    p = torch.tensor([0.1, 0.0, 0.35, 0.25, 0.3])
    q = torch.tensor([0.3, 0.2, 0.05, 0.45, 0.0])
    n = 200
    u = (torch.arange(n) + 0.5) / n
    grid = torch.cartesian_prod(u, u)
    for draft in (q, None):
        got = torch.zeros(5, dtype=torch.float64)
        for x in range(5):
            weight = float(q[x]) if draft is not None else float(x == 2)
            if weight == 0:
                continue
            R = grid.shape[0]
            coins = torch.stack([grid[:, 0], torch.zeros(R), grid[:, 1]], 1)
            acc, bonus = ops.spec_verify_probs(p.expand(R, 2, 5), None if draft is None else q.expand(R, 1, 5),
                                               torch.full((R, 1), x), coins)
            first = torch.where(acc[:, 0] == 1, torch.full((R,), x), bonus)
            got += weight * torch.bincount(first, minlength=5).double() / R
        assert (got - p.double()).abs().max() < 2 / n       # each border of the grid moves at most one cell


def test_verify_walks_the_chain():
    V, D = 6, 3
    p = torch.full((1, D + 1, V), 1.0 / V)
    q = torch.full((1, D, V), 1.0 / V)
    tok = torch.tensor([[1, 2, 3]])
    acc, bonus = ops.spec_verify_probs(p, q, tok, torch.tensor([[0.5, 0.9, 0.99, 0.3, 0.51]]))
    assert acc.tolist() == [[1, 2, 3]] and bonus.tolist() == [3]         # p = q: every draft is kept
    p[0, 1] = torch.tensor([0.5, 0.5, 0, 0, 0, 0])                       # draft 2 (token 2) has no mass
    acc, bonus = ops.spec_verify_probs(p, q, tok, torch.tensor([[0.5, 0.0, 0.0, 0.3, 0.51]]))
    assert acc.tolist() == [[1, -1, -1]] and bonus.tolist() == [1]       # residual (1/3, 1/3): 0.51 falls in the second
    acc, bonus = ops.spec_verify_probs(p, q, tok, torch.tensor([[0.5, 0.0, 0.0, 0.3, 0.51]]), torch.tensor([1], dtype=torch.int32))
    assert acc.tolist() == [[1, -1, -1]] and bonus.tolist() == [1]       # a chain of one draft: the bonus from p[1]
    acc, bonus = ops.spec_verify_probs(p[:, :1], None, torch.zeros(1, 0, dtype=torch.int64), torch.tensor([[0.0, 0.99]]))
    assert acc.shape == (1, 0) and bonus.tolist() == [5]                 # no drafts: a draw from p


def test_verify_edges():
    V = 4
    none = torch.zeros(1, 0, dtype=torch.int64)
    draw = lambda row, c: ops.spec_verify_probs(torch.tensor(row)[None, None], None, none, torch.tensor([[0.0, c]]))[1].item()  # noqa: E731
    assert draw([0.0, 0.5, 0.0, 0.5], 0.0) == 1 and draw([0.0, 0.5, 0.0, 0.5], 0.5) == 3
    assert draw([0.0] * V, 0.3) == V - 1                                 # no mass
    assert draw([float("nan"), 0.0, 1.0, 0.0], 0.9) == 2                 # NaN counts as none
    p, q = torch.tensor([[[0.5, 0.5, 0, 0]] * 2]), torch.tensor([[[0.5, 0.5, 0, 0]]])
    acc, bonus = ops.spec_verify_probs(p, q, torch.tensor([[7]]), torch.tensor([[0.1, 0.0, 0.6]]))
    assert acc.tolist() == [[-1]] and bonus.tolist() == [1]              # token outside: not kept; empty residual: from p
    acc, bonus = ops.spec_verify_probs(p, None, torch.tensor([[0]]), torch.tensor([[0.6, 0.0, 0.0]]))
    assert acc.tolist() == [[-1]] and bonus.tolist() == [1]              # greedy draft: its token is taken out


def test_verify_refusals():
    p, q = torch.rand(2, 3, 9), torch.rand(2, 2, 9)
    tok, coins = torch.zeros(2, 2, dtype=torch.int64), seeded_coins(torch.tensor([1, 2]), torch.tensor([5, 6]), 4)
    ops.spec_verify_probs(p, q, tok, coins)
    for args in ((p[:, :2], q, tok, coins), (p, q[:, :1], tok, coins), (p, q.half(), tok, coins), (p, q, tok, coins[:, :3])):
        with pytest.raises((ValueError, RuntimeError)):
            ops.spec_verify_probs(*args)
    with bounds_checks():
        ops.spec_verify_probs(p, q, tok, coins, torch.tensor([0, 2], dtype=torch.int32))
        with pytest.raises(BoundsError, match="tokens"):
            ops.spec_verify_probs(p, q, tok + 9, coins)
        with pytest.raises(BoundsError, match="coins"):
            ops.spec_verify_probs(p, q, tok, coins + 1)
        with pytest.raises(BoundsError, match="n_draft"):
            ops.spec_verify_probs(p, q, tok, coins, torch.tensor([0, 3], dtype=torch.int32))
