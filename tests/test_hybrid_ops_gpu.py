"""Chunked gated delta rule, per-head q/k norm with rotation and cache write, and verification of sampled draft chains
on the GPU, against plain implementations in 64 bits."""
import math

import pytest
import torch

from phung5_b200 import ops
from phung5_b200.engine.sampling import chain_reject_reference
from phung5_b200.ops import gdn as G

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_BF16 = 2.0 ** -8      # a bf16 rounding is off by at most half a step: eps / 2 relative to the value


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status()


# ---- gated delta rule ------------------------------------------------------------------------------------------

def _gdn_inputs(lens, hk, hv, seed=0, extra=0, kind="usual"):
    """q, k, v as slices of one projection row (strided), states at every second slot."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t, r = sum(lens) + extra, len(lens)
    conv = torch.nn.functional.silu(torch.randn(t, (2 * hk + hv) * 128 + 64, generator=gen, device=DEV)).bfloat16()
    c0, c1, c2 = hk * 128, 2 * hk * 128, (2 * hk + hv) * 128
    a = dict(q=conv[:, :c0].view(t, hk, 128), k=conv[:, c0:c1].view(t, hk, 128), v=conv[:, c1:c2].view(t, hv, 128),
             g=-torch.exp(torch.randn(t, hv, generator=gen, device=DEV) * 2 - 3), beta=torch.rand(t, hv, generator=gen, device=DEV),
             state=torch.randn(2 * r + 1, hv, 128, 128, generator=gen, device=DEV) * 0.2,
             tok_start=torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV),
             slot=(2 * torch.arange(r, dtype=torch.int32, device=DEV).flip(0) + 1), scale=1 / math.sqrt(128))
    if kind == "no decay":
        a["g"].zero_()
        a["beta"].fill_(1.0)
    elif kind == "hard decay":          # single tokens that forget nearly everything, between ones that keep it
        a["g"] = torch.where(torch.rand(t, hv, generator=gen, device=DEV) < 0.1, -3000.0, a["g"] * 0.1)
    elif kind == "resets":              # gates that close: the state starts anew there
        a["g"][::7] = float("-inf")
    elif kind == "one key":             # every token writes to the same key: the chunk's system is as dense as it gets
        a["k"].copy_(a["k"][:1].clone().expand_as(a["k"]))
        a["beta"].fill_(1.0)
        a["g"].mul_(0.01)
    elif kind == "zeros":
        a["k"][::3] = 0
        a["q"][1::3] = 0
        a["v"][2::3] = 0
        a["beta"][::5] = 0
    elif kind == "large":
        a["v"].mul_(1000)
        a["k"].mul_(100)
        a["q"].mul_(2 ** -20)
    return a


def _gdn_exact(a):
    """Token by token in fp64."""
    rep = a["v"].shape[1] // a["q"].shape[1]
    pool, out = a["state"].double(), torch.zeros(a["v"].shape, dtype=torch.float64, device=DEV)
    ts = a["tok_start"].tolist()
    unit = lambda x: (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(rep, 1)  # noqa: E731
    q, k = unit(a["q"].double()) * a["scale"], unit(a["k"].double())
    v, d, beta = a["v"].double(), a["g"].double().exp(), a["beta"].double()
    n = [ts[i + 1] - ts[i] for i in range(len(ts) - 1)]
    for step in range(max(n, default=0)):
        live = torch.tensor([i for i in range(len(n)) if n[i] > step], device=DEV)
        at, sl = a["tok_start"][live].long() + step, a["slot"][live].long()
        S = pool[sl] * d[at][..., None, None]
        vp = beta[at][..., None] * (v[at] - torch.einsum("rhij,rhi->rhj", S, k[at]))
        S = S + k[at][..., None] * vp[..., None, :]
        out[at] = torch.einsum("rhij,rhi->rhj", S, q[at])
        pool[sl] = S
    return out, pool


def _gdn_check(a, **kw):
    out, pool = _gdn_exact(a)
    got = G.gdn_chunked(**a, **kw)
    torch.cuda.synchronize()
    n = int(a["tok_start"][-1])
    # out: one bf16 rounding, on sums in fp32 whose operands carry 16 bits or more: off by at most 2^-16 of each
    # operand, five products in a row, against the largest magnitude of the head (|q^| and |k^| are at most 1)
    big = torch.maximum(out[:n].abs().amax((0, 2), keepdim=True), pool.abs().amax((0, 2, 3))[None, :, None] * a["scale"])
    assert bool(((got[:n].double() - out[:n]).abs() <= HALF_BF16 * out[:n].abs() + 2.0 ** -13 * big).all())
    # state: kept in fp32
    big = pool.abs().amax((2, 3), keepdim=True)
    assert bool(((a["state"].double() - pool).abs() <= 2.0 ** -14 * big).all())
    rel = ((a["state"].double() - pool).norm() / pool.norm()).item()
    assert rel < 1e-5, rel
    return got


@pytest.mark.parametrize("lens,hk,hv", [
    ([1], 1, 1), ([2], 4, 8), ([63], 2, 2), ([64], 2, 4), ([65], 1, 4), ([127, 129], 2, 4), ([0, 5, 0], 1, 2),
    ([128, 1, 0, 200, 17], 4, 8), ([1] * 33, 2, 4), ([8] * 20, 4, 8), ([700, 3], 1, 3), ([1500], 16, 32),
    ([300, 40, 260, 1, 77, 500], 8, 16), ([1] * 70 + [400] + [2] * 60, 2, 4), ([3] * 150, 1, 2)])
def test_gdn_chunked(lens, hk, hv):
    _gdn_check(_gdn_inputs(lens, hk, hv, seed=sum(lens) + hv))


@pytest.mark.parametrize("lens", [[200, 3, 66], [5, 9]])
def test_gdn_chunked_any_layout(lens):
    """Rows off 16-byte boundaries, heads apart, one head with a stride of its own, an output of the caller's."""
    a = _gdn_inputs(lens, 2, 4, seed=11)
    ref = _gdn_check({**a, "state": a["state"].clone()})
    t = sum(lens)
    off = {k: torch.empty(a[k].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(a[k].shape).copy_(a[k]) for k in ("q", "k", "v")}
    _gdn_check({**a, **off, "state": a["state"].clone()})
    wide = {k: torch.zeros(t, a[k].shape[1], 200, dtype=torch.bfloat16, device=DEV)[..., :128].copy_(a[k]) for k in ("q", "k", "v")}
    assert torch.equal(_gdn_check({**a, **wide, "state": a["state"].clone()}, out=torch.empty_like(ref)), ref)
    b = _gdn_inputs(lens, 1, 1, seed=12)
    one = {k: torch.as_strided(b[k].contiguous(), (t, 1, 128), (128, 1, 1)) for k in ("q", "k", "v")}
    _gdn_check({**b, **one})


@pytest.mark.parametrize("kind", ["no decay", "hard decay", "resets", "one key", "zeros", "large"])
@pytest.mark.parametrize("lens", [[200, 70], [5, 1, 9]])
def test_gdn_chunked_values(kind, lens):
    _gdn_check(_gdn_inputs(lens, 2, 4, seed=len(lens), kind=kind))


def test_gdn_chunked_long_run_equals_its_parts():
    """A run of 4200 tokens in one pass, and in three passes cut inside chunks: the state is carried in fp32."""
    a = _gdn_inputs([4200], 2, 4, seed=9)
    b = {**a, "state": a["state"].clone()}
    one = _gdn_check(a)
    parts = []
    for lo, hi in ((0, 1001), (1001, 1002), (1002, 4200)):
        cut = {k: b[k][lo:hi] for k in ("q", "k", "v", "g", "beta")}
        parts.append(G.gdn_chunked(**{**b, **cut, "tok_start": torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV)}))
    parts = torch.cat(parts).double()
    # both round the same fp32-accurate value to bf16: at most one step apart
    assert bool(((parts - one.double()).abs() <= 2 * HALF_BF16 * one.double().abs() + 2.0 ** -12 * one.double().abs().max()).all())
    assert ((a["state"] - b["state"]).norm() / a["state"].norm()).item() < 2e-5


def test_gdn_chunked_keeps_requests_apart():
    """NaN and infinities of a neighbouring request and of rows behind the last one reach no other request; rows
    behind the last one and unused slots stay as they were."""
    lens = [70, 90, 33]
    a = _gdn_inputs(lens, 2, 4, seed=3, extra=50)
    clean = {**a, "state": a["state"].clone()}
    ref = G.gdn_chunked(**clean)
    bad = {k: a[k].clone() for k in ("q", "k", "v", "g", "beta")}
    for x, val in zip(("q", "k", "v", "g", "beta"), (float("inf"), float("nan"), float("-inf"), float("nan"), float("inf"))):
        bad[x][70:160] = val
        bad[x][193:] = float("nan")
    pool = a["state"].clone()
    out = torch.full_like(a["v"].contiguous(), 5.0)
    G.gdn_chunked(**{**a, **bad, "state": pool}, out=out)
    assert torch.equal(out[:70], ref[:70]) and torch.equal(out[160:193], ref[160:193])
    assert bool((out[193:] == 5.0).all())
    for r, s in enumerate(a["slot"].tolist()):
        if r != 1:
            assert torch.equal(pool[s], clean["state"][s])
    assert torch.equal(pool[::2], a["state"][::2])


@pytest.mark.parametrize("lens", [[1] * 8, [150, 64, 9]])
def test_gdn_chunked_graph_stream_and_repeat(lens):
    """Bitwise the same eagerly, on another stream and replayed from a graph (twice, on a restored state)."""
    a = _gdn_inputs(lens, 2, 4, seed=5)
    start = a["state"].clone()
    ref = G.gdn_chunked(**a)
    end = a["state"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a["state"].copy_(start)
        other = G.gdn_chunked(**a)
    side.synchronize()
    assert torch.equal(other, ref) and torch.equal(a["state"], end)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.gdn_chunked(**a)
    for _ in range(2):
        a["state"].copy_(start)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(a["state"], end)


def test_gdn_chunked_two_streams_at_once():
    """Calls that run at the same time on two streams do not share anything."""
    sets = [_gdn_inputs([900, 200], 4, 8, seed=s) for s in (1, 2)]
    refs = [G.gdn_chunked(**{**a, "state": a["state"].clone()}) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        outs = []
        for a, st in zip(sets, streams):
            with torch.cuda.stream(st):
                outs.append(G.gdn_chunked(**{**a, "state": a["state"].clone()}))
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, refs))


def test_gdn_chunked_reports_bad_indices():
    """A slot or token range outside its buffer is skipped and reported; the other requests are done."""
    a = _gdn_inputs([20, 30, 40], 1, 2, seed=6)
    good = {**a, "state": a["state"].clone()}
    ref = G.gdn_chunked(**good)
    for key, bad in (("slot", torch.tensor([5, 7, 1], dtype=torch.int32)), ("slot", torch.tensor([5, -1, 1], dtype=torch.int32))):
        pool = a["state"].clone()
        out = G.gdn_chunked(**{**a, key: bad.to(DEV), "state": pool})
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside its buffer"):
            ops.check_status()
        assert torch.equal(out[:20], ref[:20]) and torch.equal(out[50:], ref[50:])
        assert torch.equal(pool[3], a["state"][3]) and torch.equal(pool[1], good["state"][1])
    pool = a["state"].clone()
    G.gdn_chunked(**{**a, "tok_start": torch.tensor([0, 20, 50, 91], dtype=torch.int32, device=DEV), "state": pool})
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside its buffer"):
        ops.check_status()
    assert torch.equal(pool[5], good["state"][5]) and torch.equal(pool[1], a["state"][1])


def test_gdn_chunked_refusals():
    a = _gdn_inputs([20], 2, 4)
    for key, bad in (("k", a["k"][:, :1]), ("q", a["q"].float()), ("v", a["v"][:10]), ("g", a["g"].half()),
                     ("state", a["state"].half()), ("state", a["state"][..., :64]), ("slot", a["slot"].long()),
                     ("tok_start", a["tok_start"][:1]), ("v", a["v"].transpose(0, 2)), ("slot", a["slot"].cpu()),
                     ("out", torch.empty(20, 4, 128, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            G.gdn_chunked(**{**a, key: bad})
    empty = {k: a[k][:0] for k in ("q", "k", "v", "g", "beta")}
    before = a["state"].clone()
    out = G.gdn_chunked(**{**a, **empty, "tok_start": torch.zeros(2, dtype=torch.int32, device=DEV)})
    assert out.shape == (0, 4, 128) and torch.equal(a["state"], before)


# ---- q/k norm + rotation + cache write -------------------------------------------------------------------------

def _qk_inputs(m, hq, hkv, d, rot, ps=64, seed=0, ld=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = torch.randn(m, width + ld, generator=gen, device=DEV).bfloat16()[:, :width]
    pages = m // ps + 3
    slots = torch.randperm(pages * ps, generator=gen, device=DEV)[:m]
    slots[1::5] = -1
    return dict(qkv=qkv, wq=(1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).bfloat16(),
                wk=(1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).bfloat16(), eps=1e-6,
                pos=torch.randint(0, 5000, (m,), generator=gen, device=DEV, dtype=torch.int32), slots=slots,
                cos_sin=ops.rope_table(5000, rot, 1e6, DEV),
                k_cache=torch.randn(pages, hkv, ps, d, generator=gen, device=DEV).bfloat16(),
                v_cache=torch.randn(pages, hkv, ps, d, generator=gen, device=DEV).bfloat16(), hq=hq, hkv=hkv, d=d)


def _qk_exact(a):
    """(q and k heads, v heads) in fp64, and what a last bit in fp32 is worth at each element."""
    m, hq, hkv, d, half = a["qkv"].shape[0], a["hq"], a["hkv"], a["d"], a["cos_sin"].shape[1]
    x = a["qkv"].double().reshape(m, hq + 2 * hkv, d)
    w = torch.cat([a["wq"].double().expand(hq, d), a["wk"].double().expand(hkv, d)])
    y = x[:, :hq + hkv]
    y = y / (y.square().mean(-1, keepdim=True) + a["eps"]).sqrt() * w
    c, s = a["cos_sin"].double()[a["pos"].long()][:, None].unbind(-1)
    y1, y2 = y[..., :half], y[..., half:2 * half]
    out = torch.cat([y1 * c - y2 * s, y2 * c + y1 * s, y[..., 2 * half:]], -1)
    size = torch.cat([y1.abs() + y2.abs(), y1.abs() + y2.abs(), y[..., 2 * half:].abs()], -1)
    return out, x[:, hq + hkv:], size


def _qk_check(a, **kw):
    out, v, size = _qk_exact(a)
    kc, vc = a["k_cache"].clone(), a["v_cache"].clone()
    q = ops.qk_norm_rope_kv_write(**a, **kw)
    torch.cuda.synchronize()
    hq, hkv, d, ps = a["hq"], a["hkv"], a["d"], kc.shape[2]
    # one bf16 rounding, after a sum of d squares (2^-24 each), a root and five products in fp32: below 2^-19
    tol = HALF_BF16 * out.abs() + 2.0 ** -19 * size + 1e-38
    assert bool(((q.double() - out[:, :hq]).abs() <= tol[:, :hq]).all())
    ok = a["slots"] >= 0
    s = a["slots"][ok]
    assert bool(((a["k_cache"][s // ps, :, s % ps].double() - out[ok, hq:]).abs() <= tol[ok, hq:]).all())
    kc[s // ps, :, s % ps] = a["k_cache"][s // ps, :, s % ps]
    vc[s // ps, :, s % ps] = v[ok].bfloat16()
    assert torch.equal(a["k_cache"], kc) and torch.equal(a["v_cache"], vc)      # nothing else was written
    return q


@pytest.mark.parametrize("m,hq,hkv,d,rot,ps,ld", [
    (1, 8, 2, 128, 128, 64, 0), (5, 8, 2, 128, 128, 64, 8), (37, 4, 4, 64, 64, 16, 0), (33, 16, 2, 256, 64, 64, 0),
    (129, 3, 1, 128, 32, 64, 64), (7, 1, 1, 64, 16, 1, 0), (9, 2, 1, 256, 256, 64, 0), (21, 4, 2, 128, 24, 64, 0),
    (6, 2, 2, 80, 80, 64, 0), (6, 3, 1, 96, 22, 64, 0), (4, 2, 1, 10, 6, 8, 0), (3, 2, 1, 512, 512, 64, 0),
    (17, 4, 2, 128, 128, 64, 3), (5, 3, 1, 128, 0, 64, 0), (5, 3, 1, 24, 0, 64, 0), (2000, 32, 8, 128, 128, 64, 0), (700, 64, 8, 128, 64, 64, 0)])
def test_qk_norm_rope(m, hq, hkv, d, rot, ps, ld):
    _qk_check(_qk_inputs(m, hq, hkv, d, rot, ps, seed=m + d, ld=ld))


@pytest.mark.parametrize("scale", [0.0, 1e-3, 1e4, 1e18])
def test_qk_norm_rope_values(scale):
    a = _qk_inputs(11, 4, 2, 128, 64, seed=2)
    a["qkv"].mul_(scale)
    q = _qk_check(a)
    if scale == 0:
        assert not bool(q.any())


def test_qk_norm_rope_without_cache_and_unaligned():
    a = _qk_inputs(13, 4, 2, 128, 128, seed=4)
    ref = _qk_check(a)
    none = {**a, "slots": None, "k_cache": None, "v_cache": None}
    assert torch.equal(ops.qk_norm_rope_kv_write(**none), ref)
    shifted = torch.empty(a["qkv"].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view_as(a["qkv"]).copy_(a["qkv"])
    w = torch.empty(129, dtype=torch.bfloat16, device=DEV)[1:].copy_(a["wq"])
    _qk_check({**a, "qkv": shifted, "wq": w})
    out = torch.empty(13, 4, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.qk_norm_rope_kv_write(**none, q_out=out) is out and torch.equal(out, ref)
    assert ops.qk_norm_rope_kv_write(**{**none, "qkv": a["qkv"][:0], "pos": a["pos"][:0]}).shape == (0, 4, 128)


def test_qk_norm_rope_far_rows_of_a_long_cache():
    """A cache of more than 2^31 elements: offsets pass 32 bits."""
    a = _qk_inputs(8, 2, 8, 128, 128, seed=6)
    pages = (2 ** 31) // (8 * 64 * 128) + 40
    for c in ("k_cache", "v_cache"):
        a[c] = torch.zeros(pages, 8, 64, 128, dtype=torch.bfloat16, device=DEV)
    a["slots"] = pages * 64 - 1 - 3 * torch.arange(8, device=DEV)
    out, v, size = _qk_exact(a)
    ops.qk_norm_rope_kv_write(**a)
    s = a["slots"]
    got = a["k_cache"][s // 64, :, s % 64].double()
    assert bool(((got - out[:, 2:]).abs() <= HALF_BF16 * out[:, 2:].abs() + 2.0 ** -19 * size[:, 2:]).all())
    assert torch.equal(a["v_cache"][s // 64, :, s % 64], v.bfloat16())
    assert int((a["v_cache"].view(pages, -1) != 0).any(1).sum()) == 1           # only the last page was touched


def test_qk_norm_rope_graph_and_bad_indices():
    a = _qk_inputs(19, 4, 2, 128, 128, seed=8)
    ref = ops.qk_norm_rope_kv_write(**a)
    kc = a["k_cache"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ops.qk_norm_rope_kv_write(**a)
    a["k_cache"].copy_(torch.where(kc == kc, kc, kc))
    q.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q, ref) and torch.equal(a["k_cache"], kc)
    bad = {**a, "slots": a["slots"].clone()}
    bad["slots"][0] = kc.shape[0] * 64
    ops.qk_norm_rope_kv_write(**bad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside its buffer"):
        ops.check_status()
    assert torch.equal(a["k_cache"], kc)
    bad = {**a, "pos": a["pos"].clone()}
    bad["pos"][2] = 5000
    ops.qk_norm_rope_kv_write(**bad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside its buffer"):
        ops.check_status()


def test_qk_norm_rope_refusals():
    a = _qk_inputs(5, 4, 2, 128, 128)
    for key, bad in (("qkv", a["qkv"][:, :-8]), ("qkv", a["qkv"].float()), ("wq", a["wq"][:64]), ("wk", a["wk"].float()),
                     ("pos", a["pos"].long()), ("pos", a["pos"][:4]), ("slots", a["slots"].int()), ("slots", a["slots"][:3]),
                     ("cos_sin", ops.rope_table(100, 256, 1e4, DEV)), ("k_cache", a["k_cache"][:, :1]), ("k_cache", None),
                     ("v_cache", a["v_cache"].float()), ("k_cache", a["k_cache"].transpose(1, 2)), ("pos", a["pos"].cpu()),
                     ("q_out", torch.empty(5, 4, 64, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.qk_norm_rope_kv_write(**{**a, key: bad})


# ---- verification of sampled draft chains ----------------------------------------------------------------------

def _verify_inputs(R, D, V, dtype, dense, seed=0, sharp=3.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = sharp * torch.randn(R, D + 1, V, generator=gen, device=DEV)
    p = torch.softmax(x, -1).to(dtype)
    q = torch.softmax(x[:, :D] + 0.5 * torch.randn(R, D, V, generator=gen, device=DEV), -1).to(dtype)
    tokens = torch.multinomial(q.float().reshape(-1, V).clamp(min=1e-30), 1, generator=gen).view(R, D) if dense and D else q.argmax(-1)
    return p, (q if dense else None), tokens, torch.rand(R, D + 2, generator=gen, device=DEV).clamp_(max=1 - 2 ** -24)


def _verify_check(p, q, tokens, coins, n=None):
    acc, bonus = ops.spec_verify_probs(p, q, tokens, coins, n)
    ra, rb = chain_reject_reference(p.cpu(), None if q is None else q.cpu(), tokens.cpu(), coins.cpu(), None if n is None else n.cpu())
    assert torch.equal(acc.cpu(), ra)
    assert torch.equal(bonus.cpu(), rb)
    return acc, bonus


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("R,D,V", [(1, 1, 1), (1, 4, 33), (5, 3, 1000), (3, 2, 4097), (33, 4, 511), (2, 40, 777), (4, 3, 32003),
                                   (2, 5, 128256), (300, 2, 129), (3, 0, 5000)])
def test_verify(R, D, V, dtype, dense):
    acc, _ = _verify_check(*_verify_inputs(R, D, V, dtype, dense, seed=R + D + V))
    if R == 33:
        lens = (acc >= 0).sum(1)
        assert lens.min() < lens.max()        # the inputs reach both rejected and kept drafts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_strides_and_ragged_chains(dtype):
    p, q, tokens, coins = _verify_inputs(7, 5, 2050, dtype, True, seed=3)
    wide = torch.full((7, 6, 2050 + 13), float("nan"), dtype=dtype, device=DEV)
    wide[..., 5:2055] = p
    n = torch.tensor([0, 5, 1, 3, 9, -2, 2], dtype=torch.int32, device=DEV)
    ref = _verify_check(p, q, tokens, coins, n)
    got = ops.spec_verify_probs(wide[..., 5:2055], q.transpose(0, 1).contiguous().transpose(0, 1), tokens, coins, n)
    assert all(torch.equal(x, y) for x, y in zip(got, ref))


def test_verify_edges():
    V = 3001
    p, q, tokens, coins = _verify_inputs(8, 2, V, torch.float32, True, seed=1)
    p[0, 0] = q[0, 0]                                    # the same row: always kept
    p[1, 0], q[1, 0] = 0, 0                              # no mass at all: a draw from an empty row
    p[2] = 0
    p[2, :, 2999] = 1                                    # one-hot near the end
    p[3, 0, :5] = float("nan")
    tokens[4, 0] = V                                     # outside the vocabulary
    tokens[5, 0] = -1
    p[6, 0], tokens[6, 0] = q[6, 0], V + 5               # not kept, and nothing left of p above q: a draw from p
    coins[7] = 0
    p[7, 0, tokens[7, 0]] = 0                            # 0 * q < 0 does not hold
    _verify_check(p, q, tokens, coins)
    _verify_check(p, None, tokens, coins)
    exact = torch.full((4, 1, 1024), 2.0 ** -10, device=DEV)      # sums and borders that are exact: ties go past the border
    c = torch.tensor([[0.0, 0.0], [0.0, 0.5], [0.0, 1023 / 1024], [0.0, 2.0 ** -10]], device=DEV)
    _, bonus = _verify_check(exact, None, torch.zeros(4, 0, dtype=torch.int64, device=DEV), c)
    assert bonus.tolist() == [0, 512, 1023, 1]


def test_verify_graph_and_streams():
    a = _verify_inputs(16, 4, 20011, torch.bfloat16, True, seed=2)
    ref = ops.spec_verify_probs(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.spec_verify_probs(*a)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.spec_verify_probs(*a)
    got[0].zero_()
    got[1].zero_()
    graph.replay()
    torch.cuda.synchronize()
    for x in (other, got):
        assert torch.equal(x[0], ref[0]) and torch.equal(x[1], ref[1])


def test_verify_far_rows_of_a_large_batch():
    """More than 2^31 probabilities: offsets pass 32 bits."""
    R, D, V = 70, 255, 128256
    p = torch.zeros(R, D + 1, V, dtype=torch.bfloat16, device=DEV)
    tokens = torch.randint(0, V, (R, D), device=DEV)
    p.scatter_(2, torch.cat([tokens, tokens[:, :1]], 1)[..., None], 1.0)
    acc, bonus = ops.spec_verify_probs(p, None, tokens, torch.full((R, D + 2), 0.5, device=DEV))
    assert bool((acc == torch.arange(1, D + 1, device=DEV)).all()) and torch.equal(bonus, tokens[:, 0])


def test_verify_refusals():
    p, q, tokens, coins = _verify_inputs(3, 2, 100, torch.float32, True)
    n = torch.ones(3, dtype=torch.int32, device=DEV)
    for args in ((p[:, :2], q, tokens, coins), (p, q[:, :1], tokens, coins), (p, q.half(), tokens, coins),
                 (p.double(), q.double(), tokens, coins), (p, q, tokens.int(), coins), (p, q, tokens, coins[:, :3]),
                 (p, q, tokens, coins.half()), (p, q, tokens, coins, n.long()), (p, q, tokens, coins, n[:2]),
                 (p.transpose(1, 2), q, tokens, coins), (p, q.cpu(), tokens, coins), (p, q, tokens.cpu(), coins)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.spec_verify_probs(*args)
    acc, bonus = ops.spec_verify_probs(p[:0], q[:0], tokens[:0], coins[:0])
    assert acc.shape == (0, 2) and bonus.shape == (0,)
