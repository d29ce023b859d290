"""What the serving engine's hybrid-model operators are measured on: the gated delta rule over prompts in chunks, the
per-head q/k norm with the rotation and the cache write, and the verification of sampled draft chains.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, 64 where 32 lose what matters)
or, where `own` is set, through the framework's entry points, on the same inputs.
"""
import math
import random

import torch

own = False

CHUNK = 64          # tokens per chunk of the plain chunked delta rule
EPS_L2 = 1e-6       # inside the root of the delta rule's q / k norms
EPS_RMS = 1e-6
PAGE = 64


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------

def listed():
    return [
        # gated delta rule: requests, tokens in all, key / value heads
        # the end of one short prompt on the small hybrid model's heads: latency
        {"name": "gdn 1x37 h4/8", "op": "gdn", "requests": 1, "tokens": 37, "hk": 4, "hv": 8, "ragged": False},
        # one prompt as long as a prefill pass on the small hybrid's heads: a long axis and few rows
        {"name": "gdn 1x8192 h4/8", "op": "gdn", "requests": 1, "tokens": 8192, "hk": 4, "hv": 8, "ragged": False},
        # a prefill pass of the default token budget shared by a few prompts of uneven length, larger model
        {"name": "gdn 7x8191 h16/32", "op": "gdn", "requests": 7, "tokens": 8191, "hk": 16, "hv": 32, "ragged": True},
        # a burst of short prompts admitted together
        {"name": "gdn 64x4000 h8/16", "op": "gdn", "requests": 64, "tokens": 4000, "hk": 8, "hv": 16, "ragged": True},
        # the largest pass: two budgets of tokens over many requests
        {"name": "gdn 48x16384 h16/32", "op": "gdn", "requests": 48, "tokens": 16384, "hk": 16, "hv": 32, "ragged": True},
        # q/k norm + rotation + cache write: rows, query / key heads, head size, rotated part
        # single-token steps of a few requests, small hybrid's heads
        {"name": "qkrope 5 h8/2 d128", "op": "qkrope", "rows": 5, "hq": 8, "hkv": 2, "d": 128, "rot": 128, "padded": False},
        # verification rows of a full batch, wide heads of which a quarter is rotated, padded to a graph's row count
        {"name": "qkrope 1283 h16/2 d256", "op": "qkrope", "rows": 1283, "hq": 16, "hkv": 2, "d": 256, "rot": 64, "padded": True},
        # a prefill pass of the default token budget
        {"name": "qkrope 8192 h32/8 d128", "op": "qkrope", "rows": 8192, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "padded": False},
        # draft verification: requests, drafts each, vocabulary, type of the probabilities, drafter's probabilities given
        # one request of a small vocabulary: latency
        {"name": "verify 1x4 v4096", "op": "verify", "requests": 1, "drafts": 4, "vocab": 4096, "dtype": "float32", "dense": True},
        # a full batch on a large vocabulary
        {"name": "verify 64x4 v128256", "op": "verify", "requests": 64, "drafts": 4, "vocab": 128256, "dtype": "float32", "dense": True},
        # greedy drafts (their own probabilities are one at the token), odd vocabulary, half-width probabilities
        {"name": "verify 17x7 v32003", "op": "verify", "requests": 17, "drafts": 7, "vocab": 32003, "dtype": "bfloat16", "dense": False},
        # as many requests as the engine runs
        {"name": "verify 256x5 v32000", "op": "verify", "requests": 256, "drafts": 5, "vocab": 32000, "dtype": "bfloat16", "dense": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gdn", "qkrope", "verify"])
    if op == "gdn":
        hk, ratio = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 2, 4])
        hv = min(hk * ratio, 32)
        tokens = min(_log(rng, 20, 16384), 16384 * 32 // hv)
        return {"op": op, "requests": min(_log(rng, 1, 48), tokens), "tokens": tokens, "hk": hk, "hv": hv,
                "ragged": rng.random() < 0.8}
    if op == "qkrope":
        hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        d = rng.choice([64, 128, 128, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        rows = _log(rng, 1, max(2, 8192 * 48 * 128 // ((hkv * group + 2 * hkv) * d)))
        return {"op": op, "rows": min(rows, 16384), "hq": hkv * group, "hkv": hkv, "d": d, "rot": rot,
                "padded": rng.random() < 0.5}
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    drafts = rng.randint(1, 8)
    vocab = _log(rng, 1000, 152064)
    requests = min(_log(rng, 1, 256), max(1, 64 * 4 * 128256 // (vocab * drafts)))
    return {"op": op, "requests": requests, "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "dense": rng.random() < 0.7}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------

def _lens(case, seed):
    """Token counts of the requests: equal, or uneven by a log-normal share (one of many may get none)."""
    r, t = case["requests"], case["tokens"]
    rng = random.Random(seed * 7919 + 1)
    share = [math.exp(rng.gauss(0.0, 1.0)) if case["ragged"] else 1.0 for _ in range(r)]
    total, acc, cuts = sum(share), 0.0, [0]
    for s in share:
        acc += s
        cuts.append(int(round(acc / total * t)))
    cuts[-1] = t
    return [b - a for a, b in zip(cuts, cuts[1:])]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "gdn":
        lens, hk, hv = _lens(case, seed), case["hk"], case["hv"]
        r, t = len(lens), case["tokens"]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        # the layer's convolution output [q | k | v] (SiLU of a sum over taps), its gates (decay rates from a
        # model's usual initialisation: time constants of one to a thousand tokens) and a state pool in use
        conv = torch.nn.functional.silu(randn(t, (2 * hk + hv) * 128)).to(torch.bfloat16)
        rate = 1.0 + 15.0 * torch.rand(hv, generator=gen, device=dev)
        step = torch.exp(math.log(1e-3) + torch.rand(hv, generator=gen, device=dev) * math.log(100.0))
        bias = step + torch.log(-torch.expm1(-step))
        a, b = randn(t, hv).to(torch.bfloat16), randn(t, hv).to(torch.bfloat16)
        g = -rate * torch.nn.functional.softplus(a.float() * 0.5 + bias)
        order = list(range(r + 2))
        random.Random(seed + 5).shuffle(order)
        pool = randn(r + 2, hv, 128, 128) * 0.2
        k0, v0 = hk * 128, 2 * hk * 128
        return {"case": case, "lens": lens, "starts": starts, "slots": order[:r],
                "q": conv[:, :k0].view(t, hk, 128), "k": conv[:, k0:v0].view(t, hk, 128), "v": conv[:, v0:].view(t, hv, 128),
                "g": g, "beta": torch.sigmoid(b.float()), "state": pool, "scale": 1.0 / math.sqrt(128),
                "tok_start": torch.tensor(starts, dtype=torch.int32, device=dev),
                "slot": torch.tensor(order[:r], dtype=torch.int32, device=dev)}

    if case["op"] == "qkrope":
        m, hq, hkv, d, rot = case["rows"], case["hq"], case["hkv"], case["d"], case["rot"]
        qkv = (randn(m, (hq + 2 * hkv) * d) * 1.5).to(torch.bfloat16)
        pages = 2 * ((m + PAGE - 1) // PAGE) + 1
        page = torch.randperm(pages, generator=gen, device=dev)
        row = torch.arange(m, device=dev)
        slots = page[row // PAGE] * PAGE + row % PAGE
        if case["padded"]:      # rows behind the batch's last token write nothing to the cache
            slots[m - m // 8:] = -1
        cache = [randn(pages, hkv, PAGE, d).to(torch.bfloat16) for _ in range(2)]
        max_pos = 16384
        inv = 1e7 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        ang = torch.arange(max_pos, dtype=torch.float64, device=dev)[:, None] * inv
        first = torch.randint(0, max_pos - m + 1 if m < max_pos else 1, (1,), generator=gen, device=dev)
        return {"case": case, "qkv": qkv, "wq": (1 + 0.2 * randn(d)).to(torch.bfloat16),
                "wk": (1 + 0.2 * randn(d)).to(torch.bfloat16), "pos": (first + row).to(torch.int32), "slots": slots,
                "cos_sin": torch.stack([ang.cos(), ang.sin()], -1).float(), "k_cache": cache[0], "v_cache": cache[1]}

    r, n, v, dt = case["requests"], case["drafts"], case["vocab"], getattr(torch, case["dtype"])
    # target and draft distributions that mostly agree, peaked as a language model's; drafts drawn from the
    # drafter's distribution (or its largest value where drafts are greedy)
    target = 3.0 * randn(r, n + 1, v)
    p = torch.softmax(target, -1).to(dt)
    q = torch.softmax(target[:, :n] + 0.4 * randn(r, n, v), -1).to(dt)
    del target
    if case["dense"]:
        race = torch.rand(r, n, v, generator=gen, device=dev).clamp_(min=1e-20).log_().neg_()
        tokens = (q.float() / race).argmax(-1)
        del race
    else:
        tokens = q.argmax(-1)
        q = None
    return {"case": case, "p": p, "q": q, "tokens": tokens,
            "coins": torch.rand(r, n + 2, generator=gen, device=dev).clamp_(max=1 - 2 ** -24)}


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "gdn":
        return _gdn_own(state) if own else _gdn_plain(state)
    if op == "qkrope":
        return _qkrope_own(state) if own else _qkrope_plain(state)
    return _verify_own(state) if own else _verify_plain(state)


def _gdn_own(s):
    from phung5_b200.ops import gdn as G
    out = G.gdn_chunked(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["tok_start"], s["slot"], s["scale"])
    return {"out": out, "state": s["state"]}


def _qkrope_own(s):
    from phung5_b200 import ops
    c = s["case"]
    q = ops.qk_norm_rope_kv_write(s["qkv"], s["wq"], s["wk"], EPS_RMS, s["pos"], s["slots"], s["cos_sin"], s["k_cache"],
                                  s["v_cache"], c["hq"], c["hkv"], c["d"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _verify_own(s):
    from phung5_b200 import ops
    accepted, bonus = ops.spec_verify_probs(s["p"], s["q"], s["tokens"], s["coins"])
    return {"accepted": accepted, "bonus": bonus}


def _gdn_plain(s):
    """Chunks of 64 tokens: everything inside a chunk for all chunks at once, then the chunks of all requests in step."""
    hk, hv, dev = s["case"]["hk"], s["case"]["hv"], s["q"].device
    rep = hv // hk
    lens = torch.tensor(s["lens"])
    order = torch.argsort(lens, descending=True)
    lens, start = lens[order], torch.tensor(s["starts"][:-1])[order]
    slot = s["slot"][order.to(dev)].long()
    most = (int(lens[0]) + CHUNK - 1) // CHUNK
    # chunk c of every request that has one, c by c; requests from the longest to the shortest
    c, r = torch.nonzero(torch.arange(most)[:, None] * CHUNK < lens, as_tuple=True)
    counts = torch.bincount(c, minlength=most).tolist()
    tok = (start[r] + c * CHUNK)[:, None] + torch.arange(CHUNK)
    here = (torch.arange(CHUNK) < (lens[r] - c * CHUNK)[:, None]).to(dev)
    tok = tok.clamp(max=s["q"].shape[0] - 1).to(dev)

    def unit(x):
        x = x.float()
        return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS_L2)

    def rows(x):        # [T, H, ...] -> [chunks, H, 64, ...], zero past a request's end
        x = x[tok]
        return torch.where(here.view(here.shape + (1,) * (x.dim() - 2)), x, 0.0).transpose(1, 2)

    Q, K = rows(unit(s["q"]) * s["scale"]), rows(unit(s["k"]))
    V, beta = rows(s["v"].float()), rows(s["beta"])
    b = rows(s["g"].double()).cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=dev).tril()
    decay = torch.where(low, torch.exp(torch.where(low, b[..., :, None] - b[..., None, :], 0.0)), 0.0).float()
    grow, keep = torch.exp(b).float(), torch.exp(b[..., -1:] - b).float()
    KK = (K @ K.transpose(-1, -2)).repeat_interleave(rep, 1)
    P = (Q @ K.transpose(-1, -2)).repeat_interleave(rep, 1) * decay
    L = (KK * decay * beta[..., None]).tril(-1)
    T = torch.eye(CHUNK, device=dev).expand_as(L).clone()
    for i in range(1, CHUNK):
        T[..., i, :i] = -(L[..., i:i + 1, :i] @ T[..., :i, :i])[..., 0, :]
    Q, K = Q.repeat_interleave(rep, 1), K.repeat_interleave(rep, 1)
    S = s["state"][slot]
    O = torch.empty_like(V)
    at = 0
    for n in counts:
        u, S0 = slice(at, at + n), S[:n]
        e = grow[u][..., None]
        X = T[u] @ (beta[u][..., None] * (V[u] - e * (K[u] @ S0)))
        O[u] = e * (Q[u] @ S0) + P[u] @ X
        S[:n] = S0 * e[..., -1:, :] + (K[u] * keep[u][..., None]).transpose(-1, -2) @ X
        at += n
    out = torch.empty(s["v"].shape, dtype=torch.bfloat16, device=dev)
    out[tok[here]] = O.transpose(1, 2)[here].to(torch.bfloat16)
    s["state"][slot] = S
    return {"out": out, "state": s["state"]}


def _qkrope_plain(s):
    c = s["case"]
    m, hq, hkv, d, rot = c["rows"], c["hq"], c["hkv"], c["d"], c["rot"]
    x = s["qkv"].float().view(m, hq + 2 * hkv, d)
    w = torch.cat([s["wq"].float().expand(hq, d), s["wk"].float().expand(hkv, d)])
    y = x[:, :hq + hkv]
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS_RMS) * w
    cos, sin = s["cos_sin"][s["pos"].long()][:, None].unbind(-1)
    y1, y2 = y[..., :rot // 2], y[..., rot // 2:rot]
    y = torch.cat([y1 * cos - y2 * sin, y2 * cos + y1 * sin, y[..., rot:]], -1).to(torch.bfloat16)
    kept = s["slots"] >= 0
    slot = s["slots"][kept]
    s["k_cache"][slot // PAGE, :, slot % PAGE] = y[kept, hq:]
    s["v_cache"][slot // PAGE, :, slot % PAGE] = x[kept, hq + hkv:].to(torch.bfloat16)
    return {"q": y[:, :hq].contiguous(), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _verify_plain(s):
    p, q, tokens, coins = s["p"], s["q"], s["tokens"], s["coins"]
    r, n = tokens.shape
    rows = torch.arange(r, device=p.device)
    px = p[:, :n].gather(2, tokens[..., None])[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(2, tokens[..., None])[..., 0].double()
    kept = (coins[:, :n].double() * qx < px).long().cumprod(1)
    accepted = kept.sum(1)
    last = p[rows, accepted].double()
    at = accepted.clamp(max=n - 1)
    if q is None:
        other = torch.zeros_like(last).scatter_(1, tokens[rows, at][:, None], 2.0)
    else:
        other = q[rows, at].double()
    rest = torch.where((accepted == n)[:, None], last, (last - other).clamp(min=0))
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, last)
    mass = rest.cumsum(1)
    bonus = (mass <= coins[:, n + 1:].double() * mass[:, -1:]).sum(1).clamp(max=p.shape[2] - 1)
    node = torch.arange(1, n + 1, device=p.device).expand(r, n)
    return {"accepted": torch.where(kept > 0, node, -1), "bonus": bonus}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gdn":
        return _gdn_exact(s)
    if case["op"] == "qkrope":
        return _qkrope_exact(s)
    return _verify_exact(s)


def _gdn_exact(s):
    """Token by token, every request that still has one in each step."""
    lens, dev = s["lens"], s["q"].device
    rep = s["case"]["hv"] // s["case"]["hk"]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    start = torch.tensor([s["starts"][i] for i in order], device=dev)
    slot = torch.tensor([s["slots"][i] for i in order], device=dev)
    pool = s["state"].double()
    S = pool[slot]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=dev)
    n = len(order)
    for t in range(lens[order[0]]):
        while lens[order[n - 1]] <= t:
            n -= 1
        at = start[:n] + t
        q, k = s["q"][at].double(), s["k"][at].double()
        q = (q / (q.square().sum(-1, keepdim=True) + EPS_L2).sqrt() * s["scale"]).repeat_interleave(rep, 1)
        k = (k / (k.square().sum(-1, keepdim=True) + EPS_L2).sqrt()).repeat_interleave(rep, 1)
        M = S[:n].mul_(s["g"][at].double().exp()[..., None, None])
        new = s["beta"][at].double()[..., None] * (s["v"][at].double() - torch.einsum("rhij,rhi->rhj", M, k))
        M += k[..., :, None] * new[..., None, :]
        out[at] = torch.einsum("rhij,rhi->rhj", M, q)
    pool[slot] = S
    return {"out": out, "state": pool}


def _qkrope_exact(s):
    c = s["case"]
    m, hq, hkv, d, half = c["rows"], c["hq"], c["hkv"], c["d"], c["rot"] // 2
    q, k, v = s["qkv"].double().split([hq * d, hkv * d, hkv * d], 1)
    table = s["cos_sin"].double()[s["pos"].long()]
    turn = torch.complex(table[..., 0], table[..., 1])[:, None]

    def head(x, w):
        x = x.view(m, -1, d)
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS_RMS).sqrt() * w.double()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    caches = []
    for cache, x in ((s["k_cache"], head(k, s["wk"])), (s["v_cache"], v.view(m, hkv, d))):
        flat = cache.double().transpose(1, 2).reshape(-1, hkv, d)
        use = torch.nonzero(s["slots"] >= 0)[:, 0]
        flat[s["slots"][use]] = x[use]
        caches.append(flat.view(-1, PAGE, hkv, d).transpose(1, 2).contiguous())
    return {"q": head(q, s["wq"]), "k_cache": caches[0], "v_cache": caches[1]}


def _verify_exact(s):
    """Request by request on the host."""
    p, q, tokens, coins = s["p"], s["q"], s["tokens"].tolist(), s["coins"].double().cpu()
    accepted, bonus = [], []
    for r, drafts in enumerate(tokens):
        kept = 0
        for j, x in enumerate(drafts):
            if float(coins[r, j]) * (1.0 if q is None else float(q[r, j, x])) >= float(p[r, j, x]):
                break
            kept += 1
        rest = p[r, kept].double()
        if kept < len(drafts):
            if q is None:
                cut = rest.clone()
                cut[drafts[kept]] = 0
            else:
                cut = torch.relu(rest - q[r, kept].double())
            rest = cut if float(cut.sum()) > 0 else rest
        mass = torch.cumsum(rest, 0)
        bonus.append(int(torch.searchsorted(mass, coins[r, -1].to(mass.device) * mass[-1], right=True)))
        accepted.append([j + 1 if j < kept else -1 for j in range(len(drafts))])
    dev = p.device
    return {"accepted": torch.tensor(accepted, device=dev), "bonus": torch.tensor(bonus, device=dev).clamp(max=p.shape[2] - 1)}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "gdn":
        t, hk, hv, r = case["tokens"], case["hk"], case["hv"], case["requests"]
        per_head = 3 * 2 * 128 * 128 + 4 * 2 * CHUNK * 128      # state products, and products inside a chunk
        return {"bytes": t * (2 * (2 * hk + 2 * hv) * 128 + 2 * hv * 4) + r * (2 * hv * 128 * 128 * 4 + 8),
                "flops": t * hv * per_head}
    if case["op"] == "qkrope":
        m, hq, hkv, d, rot = case["rows"], case["hq"], case["hkv"], case["d"], case["rot"]
        return {"bytes": m * (2 * 2 * (hq + 2 * hkv) * d + 4 * rot + 12) + 4 * d, "flops": m * (hq + hkv) * (4 * d + 3 * rot)}
    size = 4 if case["dtype"] == "float32" else 2
    r, n, v = case["requests"], case["drafts"], case["vocab"]
    # one row of the target's (and of the drafter's) probabilities for each request, and each draft's own values
    return {"bytes": r * ((2 if case["dense"] else 1) * v * size + n * (8 + 4 + 2 * size) + 8 * (n + 2)),
            "flops": r * v * (2 if case["dense"] else 1)}
