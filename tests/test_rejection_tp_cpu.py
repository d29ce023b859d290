"""Sampled draft chains verified by rejection on two gloo ranks (vocabulary in shards)."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from phung5_b200.config import CacheConfig, DraftConfig, EngineConfig, SpecConfig, preset


def _worker(rank, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        from phung5_b200.engine import engine as E
        from phung5_b200.engine.oracle import SamplingParams
        from phung5_b200.models.llama import pack_weights
        from phung5_b200.parallel.comm import NcclCommunicator
        from phung5_b200.weights.init import random_weights
        tcfg, dcfg = preset("tiny"), preset("tiny-draft")
        E._DraftSampler.PIECE = 3 * tcfg.vocab           # pieces of three rows: 3 x 4 rows to verify, two requests left at the end
        cfg = EngineConfig(model=tcfg, spec=SpecConfig(mode="chain", num_draft=3, accept="rejection"), draft=DraftConfig(kind="model"),
                           cache=CacheConfig(page_size=16, num_pages=200))
        w = [pack_weights(c, random_weights(c, seed=s, std=0.05), "cpu", rank, 2, dtype=torch.float32) for s, c in enumerate((tcfg, dcfg))]
        eng = E.LLMEngine(cfg, device="cpu", target=w[0], drafter=w[1], comm=NcclCommunicator(), dtype=torch.float32, max_context=512)
        rids = [eng.add_request([7, 8, 9, 10 + i], SamplingParams(max_new_tokens=n, temperature=t, top_k=20, seed=i))
                for i, (n, t) in enumerate(((9, 0.8), (4, 0.0), (9, 1.2)))]
        while eng.has_work():
            eng.step()
        q.put((rank, [eng.reqs[r].out for r in rids], eng.stats["spec_steps"]))
    finally:
        dist.destroy_process_group()


def test_ranks_take_the_same_pieces_and_the_same_tokens():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    procs = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=240) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    assert all(p.exitcode == 0 for p in procs)
    assert res[0][1:] == res[1][1:] and [len(o) for o in res[0][1]] == [9, 4, 9] and res[0][2] > 0
